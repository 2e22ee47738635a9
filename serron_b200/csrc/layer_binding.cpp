// The layer operators as torch sees them: outputs and workspaces from torch's caching allocator, work on torch's
// current stream, and backward nodes that call the C ABI (include/serron_b200.h) without passing through Python.
//
// A pass of these operators over a small tensor takes a few microseconds on the GPU, and a custom function written in
// Python about forty on the host, forward and backward; from here the two passes cost a few each.  Arguments are
// checked by the Python functions (serron_b200/functional.py) before they come here.
#include "serron_b200.h"

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
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
Tensor plain(const MaybeTensor& t) { return t.has_value() && t->defined() ? t->contiguous() : Tensor(); }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int32_t ordinal_of(const Tensor& t) { return t.device().index(); }

// How the memory of a dense tensor holds the rows along `dim`.
struct Layout {
    int64_t outer = 1, len = 1, inner = 1;
};

// The layout of x; x becomes a contiguous copy where its dimensions do not lie densely in some order.
Layout layout_of(Tensor& x, int64_t dim) {
    const int64_t n = x.dim();
    c10::SmallVector<int64_t, 8> order(n);
    std::iota(order.begin(), order.end(), 0);
    if (!x.is_contiguous()) {
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
    }
    Layout l;
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

struct Workspace {
    Tensor buffer;
    int64_t bytes;
    Workspace(const Tensor& x, const Layout& l, bool backward)
        : bytes(serron_layer_norm_workspace_bytes(l.outer, l.len, l.inner, dtype_code(x.scalar_type()), backward)) {
        if (bytes < 0) raise_for(SERRON_ERR_INVALID);
        if (bytes > 0) buffer = at::empty({bytes}, x.options().dtype(at::kByte));
    }
};

// mean in the first row, 1 / sqrt(var + eps) in the second
Tensor empty_stats(const Tensor& x, const Layout& l) {
    return at::empty({2, l.outer * l.inner},
                     x.options().dtype(x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat));
}
void* second(const Tensor& stats) {
    return stats.defined() ? static_cast<char*>(stats.data_ptr()) + stats.size(1) * stats.element_size() : nullptr;
}

struct Rule {
    double p = 0.0;
    uint64_t seed = 0, sequence = 0;
};

at::ScalarType param_type(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    return weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : x.scalar_type();
}

// Gradients of a backward pass cannot be differentiated again: where a graph of them is asked for, its use is an error.
variable_list once(variable_list&& grads) {
    if (!at::GradMode::is_enabled()) return std::move(grads);
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    torch::autograd::DelayedError error(
        "serron: a gradient of layer_norm, dropout or dropout_add_layer_norm is once_differentiable",
        static_cast<int64_t>(grads.size()));
    return error.apply(std::move(grads));
}

// ------------------------------------------------------------------------------------------------
// layer norm
// ------------------------------------------------------------------------------------------------
struct LayerNormBackward : public Node {
    SavedVariable x, weight, stats;
    Layout layout;
    at::ScalarType params = at::kFloat;

    std::string name() const override { return "SerronLayerNormBackward"; }
    void release_variables() override {
        x.reset_data();
        weight.reset_data();
        stats.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        if (!grads[0].defined()) return variable_list(3);
        variable_list out(3);
        {
            at::NoGradGuard no_grad;
            const Tensor input = x.unpack(), w = plain(weight.unpack()), s = stats.unpack();
            const Tensor gy = like(grads[0], input);
            if (task_should_compute_output(0)) out[0] = at::empty_like(input);
            for (const int i : {1, 2})
                if (task_should_compute_output(i)) out[i] = at::empty({layout.len}, input.options().dtype(params));
            const Workspace ws(input, layout, true);
            raise_for(serron_layer_norm_backward(
                address(gy), address(input), address(s), second(s), layout.outer, layout.len, layout.inner,
                dtype_code(input.scalar_type()), address(w), dtype_code(params), address(out[0]), address(out[1]),
                address(out[2]), address(ws.buffer), ws.bytes, ordinal_of(input), stream_of(input)));
        }
        return once(std::move(out));
    }
};

Tensor layer_norm(const Tensor& input, const MaybeTensor& weight, const MaybeTensor& bias, int64_t dim, double eps) {
    const Tensor none;
    const Tensor &given_w = weight.has_value() ? *weight : none, &given_b = bias.has_value() ? *bias : none;
    const bool records = torch::autograd::compute_requires_grad(input, given_w, given_b);
    Tensor x = input, y, stats;
    Layout layout;
    at::ScalarType params;
    {
        at::NoGradGuard no_grad;
        layout = layout_of(x, dim);
        const Tensor w = plain(weight), b = plain(bias);
        params = param_type(x, w, b);
        y = at::empty_like(x);
        if (records) stats = empty_stats(x, layout);
        const Workspace ws(x, layout, false);
        raise_for(serron_layer_norm(address(x), layout.outer, layout.len, layout.inner, dtype_code(x.scalar_type()),
                                    address(w), address(b), dtype_code(params), eps, address(y), address(stats),
                                    second(stats), address(ws.buffer), ws.bytes, ordinal_of(x), stream_of(x)));
    }
    if (records) {
        auto node = std::make_shared<LayerNormBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(input, given_w, given_b));
        node->x = SavedVariable(x, false);
        node->weight = SavedVariable(given_w, false);
        node->stats = SavedVariable(stats, false);
        node->layout = layout;
        node->params = params;
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ------------------------------------------------------------------------------------------------
// dropout
// ------------------------------------------------------------------------------------------------
Tensor run_dropout(const Tensor& x, const Tensor& residual, int64_t span, const Rule& rule, const Tensor& seed) {
    Tensor y = at::empty_like(x);
    raise_for(serron_dropout(address(x), address(residual), x.numel(), span, dtype_code(x.scalar_type()), rule.p,
                             rule.seed, address(seed), rule.sequence, address(y), ordinal_of(x), stream_of(x)));
    return y;
}

struct DropoutBackward : public Node {
    SavedVariable seed;
    Rule rule;
    int64_t span = 1;

    std::string name() const override { return "SerronDropoutBackward"; }
    void release_variables() override { seed.reset_data(); }

    variable_list apply(variable_list&& grads) override {
        if (!grads[0].defined()) return variable_list(2);
        variable_list out(2);
        {
            at::NoGradGuard no_grad;
            if (task_should_compute_output(0))
                out[0] = run_dropout(grads[0].contiguous(), Tensor(), span, rule, seed.unpack());
        }
        out = once(std::move(out));
        if (task_should_compute_output(1)) out[1] = grads[0];
        return out;
    }
};

Tensor dropout(const Tensor& input, const MaybeTensor& residual, int64_t span, double p, uint64_t seed,
               const MaybeTensor& seed_tensor, uint64_t sequence) {
    const Tensor none;
    const Tensor& given_r = residual.has_value() ? *residual : none;
    const Rule rule{p, seed, sequence};
    const bool records = torch::autograd::compute_requires_grad(input, given_r);
    Tensor y;
    {
        at::NoGradGuard no_grad;
        y = run_dropout(input.contiguous(), plain(residual), span, rule, seed_tensor.value_or(Tensor()));
    }
    if (records) {
        auto node = std::make_shared<DropoutBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(input, given_r));
        node->seed = SavedVariable(seed_tensor.value_or(Tensor()), false);
        node->rule = rule;
        node->span = span;
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ------------------------------------------------------------------------------------------------
// the join
// ------------------------------------------------------------------------------------------------
struct DropoutAddLayerNormBackward : public Node {
    SavedVariable sum, weight, stats, seed;
    Layout layout;
    Rule rule;
    at::ScalarType params = at::kFloat;

    std::string name() const override { return "SerronDropoutAddLayerNormBackward"; }
    void release_variables() override {
        sum.reset_data();
        weight.reset_data();
        stats.reset_data();
        seed.reset_data();
    }

    variable_list apply(variable_list&& grads) override {
        if (!grads[0].defined() && !grads[1].defined()) return variable_list(4);
        variable_list out(4);
        {
            at::NoGradGuard no_grad;
            const Tensor h = sum.unpack(shared_from_this()), w = plain(weight.unpack()), s = stats.unpack();
            const Tensor key = seed.unpack();
            const Tensor gy = grads[0].defined() ? like(grads[0], h) : at::zeros_like(h);
            const Tensor gh = grads[1].defined() ? like(grads[1], h) : Tensor();
            for (const int i : {0, 1})
                if (task_should_compute_output(i)) out[i] = at::empty_like(h);
            for (const int i : {2, 3})
                if (task_should_compute_output(i)) out[i] = at::empty({layout.len}, h.options().dtype(params));
            const Workspace ws(h, layout, true);
            raise_for(serron_dropout_add_layer_norm_backward(
                address(gy), address(gh), address(h), address(s), second(s), layout.outer, layout.len, layout.inner,
                dtype_code(h.scalar_type()), address(w), dtype_code(params), rule.p, rule.seed, address(key),
                rule.sequence, address(out[0]), address(out[1]), address(out[2]), address(out[3]), address(ws.buffer),
                ws.bytes, ordinal_of(h), stream_of(h)));
        }
        return once(std::move(out));
    }
};

std::tuple<Tensor, Tensor> dropout_add_layer_norm(const Tensor& input, const Tensor& residual, const MaybeTensor& weight,
                                                  const MaybeTensor& bias, double p, uint64_t seed,
                                                  const MaybeTensor& seed_tensor, uint64_t sequence, int64_t dim,
                                                  double eps) {
    const Tensor none;
    const Tensor &given_w = weight.has_value() ? *weight : none, &given_b = bias.has_value() ? *bias : none;
    const Tensor key = seed_tensor.value_or(Tensor());
    const Rule rule{p, seed, sequence};
    const bool records = torch::autograd::compute_requires_grad(input, residual, given_w, given_b);
    Tensor y, h, stats;
    Layout layout;
    at::ScalarType params;
    {
        at::NoGradGuard no_grad;
        Tensor x = input.contiguous();  // decisions are counted in the row-major order of the elements
        const Tensor r = residual.contiguous(), w = plain(weight), b = plain(bias);
        layout = layout_of(x, dim);
        params = param_type(x, w, b);
        y = at::empty_like(x);
        h = at::empty_like(x);
        if (records) stats = empty_stats(x, layout);
        const Workspace ws(x, layout, false);
        raise_for(serron_dropout_add_layer_norm(
            address(x), address(r), layout.outer, layout.len, layout.inner, dtype_code(x.scalar_type()), address(w),
            address(b), dtype_code(params), p, seed, address(key), sequence, eps, address(h), address(y),
            address(stats), second(stats), address(ws.buffer), ws.bytes, ordinal_of(x), stream_of(x)));
    }
    if (records) {
        auto node = std::make_shared<DropoutAddLayerNormBackward>();
        node->set_next_edges(torch::autograd::collect_next_edges(input, residual, given_w, given_b));
        torch::autograd::set_history(y, node);
        torch::autograd::set_history(h, node);
        node->sum = SavedVariable(h, true);
        node->weight = SavedVariable(given_w, false);
        node->stats = SavedVariable(stats, false);
        node->seed = SavedVariable(key, false);
        node->layout = layout;
        node->rule = rule;
        node->params = params;
    }
    return {y, h};
}

}  // namespace

PYBIND11_MODULE(_layers, m) {
    m.doc() = "Layer norm, dropout and their join over the C ABI, with their backward nodes.";
    m.def("layer_norm", &layer_norm);
    m.def("dropout", &dropout);
    m.def("dropout_add_layer_norm", &dropout_add_layer_norm);
}
