// What shared codes and tokens are learned with, for Python: the cross entropy of rows against a table, dropout and the balance
// loss as C++ autograd functions.
#include <torch/csrc/utils/pybind.h>

#include <cmath>

#include "torch_common.h"

namespace py = pybind11;

namespace efgs_torch {

namespace {

void check_dense(const char* name, const Tensor& t, at::Device device) {
    TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.device().is_cuda(), "efgs: ", name, " must be a dense tensor on a GPU device, got ", t.layout(),
                      " on ", t.device());
    TORCH_CHECK_VALUE(t.device() == device, "efgs: ", name, " are on ", t.device(), ", expected ", device);
}

void check_index_type(const char* name, const Tensor& t) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, "efgs: ", name, " must be int32 or int64, got ", t.dtype());
}

// (an evaluation that needs no graph passes the autograd function by, which would refuse: its result would have lost the tangent)
void check_no_tangent(const char* name, const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(), "efgs: ", name, " has no forward-mode derivative");
}

bool needs_graph(const Tensor& t) { return at::GradMode::is_enabled() && t.defined() && t.requires_grad(); }

// a float32 upstream gradient of `n` values on the device (a node called directly is given whatever its caller has)
Tensor float_upstream(const Tensor& upstream, int64_t n, at::Device device) {
    TORCH_CHECK_VALUE(upstream.scalar_type() == at::kFloat && upstream.numel() == n && upstream.device() == device,
                      "efgs: the loss's gradient must hold ", n, " float32 values on ", device);
    return upstream.contiguous();
}

// ---- cross entropy against the rows of a table ---------------------------------------------------------------------------

efgs_entropy entropy_of(const Tensor& table, int64_t n, int32_t reduction, double scale) {
    efgs_entropy e{};
    e.table = pointer<void>(table);
    e.n = n;
    e.rows = table.size(0);
    e.columns = table.size(1);
    e.feature_stride = e.columns;
    e.table_stride = e.rows > 1 ? table.stride(0) : e.columns;
    e.target_bytes = 8;
    e.type = element_type("the table", table.scalar_type());
    e.reduction = reduction;
    e.scale = static_cast<float>(scale);
    return e;
}

// a table as the kernels read it: rows of consecutive elements
Tensor rows_of(const Tensor& t) { return t.size(1) > 1 && t.stride(1) != 1 ? t.contiguous() : t; }

struct EntropyCall {
    Tensor features, targets;   // (n, columns), n
    int64_t n = 0;
    int32_t reduction = EFGS_MEAN;
    double scale = 1.0;
};

Tensor entropy_forward(const EntropyCall& c, const Tensor& table, void* saved) {
    const at::Device device = table.device();
    const Tensor w = rows_of(table);
    efgs_entropy e = entropy_of(w, c.n, c.reduction, c.scale);
    e.features = pointer<void>(c.features);
    e.targets = pointer<void>(c.targets);
    e.feature_stride = c.n > 1 ? c.features.stride(0) : e.columns;
    e.target_bytes = static_cast<int32_t>(c.targets.element_size());
    const auto options = at::TensorOptions().dtype(at::kFloat).device(device);
    const Tensor loss = c.reduction == EFGS_EACH ? at::empty(c.targets.sizes(), options) : at::empty({}, options);
    Scratch scratch(device);
    check_status(efgs_linear_cross_entropy_forward(&e, pointer<float>(loss), saved, &Scratch::alloc, &scratch, current_stream(device)));
    return loss;
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
    static Tensor forward(AutogradContext* ctx, const Tensor& features, const Tensor& table, const EntropyCall& c) {
        const Tensor w = table.detach();
        const efgs_entropy e = entropy_of(w, c.n, c.reduction, c.scale);
        const int64_t bytes = efgs_linear_cross_entropy_saved_bytes(&e);
        if (bytes < 0) check_status(EFGS_ERR_INVALID_ARGUMENT);
        const Tensor saved = at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(table.device()));
        const Tensor loss = entropy_forward(c, w, saved.data_ptr());
        ctx->saved_data["shape"] = features.sizes();
        ctx->saved_data["n"] = c.n;
        ctx->saved_data["reduction"] = static_cast<int64_t>(c.reduction);
        ctx->saved_data["scale"] = c.scale;
        ctx->save_for_backward({table, saved});
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list grads(3);
        {
            at::NoGradGuard no_grad;
            const at::Device device = saved[0].device();
            const c10::DeviceGuard guard(device);
            const Tensor table = rows_of(saved[0].detach());
            const int64_t n = ctx->saved_data["n"].toInt();
            const auto reduction = static_cast<int32_t>(ctx->saved_data["reduction"].toInt());
            const efgs_entropy e = entropy_of(table, n, reduction, ctx->saved_data["scale"].toDouble());
            TORCH_CHECK_VALUE(saved[1].device() == device && saved[1].scalar_type() == at::kByte && saved[1].is_contiguous() &&
                                  saved[1].numel() == efgs_linear_cross_entropy_saved_bytes(&e),
                              "efgs: the cross entropy's saved rows are not what its forward saved");
            const Tensor g = float_upstream(upstream[0], reduction == EFGS_EACH ? n : 1, device);
            if (ctx->needs_input_grad(0)) grads[0] = at::empty(ctx->saved_data["shape"].toIntVector(), table.options());
            if (ctx->needs_input_grad(1)) grads[1] = at::empty({e.rows, e.columns}, table.options());
            Scratch scratch(device);
            check_status(efgs_linear_cross_entropy_backward(&e, pointer<float>(g), saved[1].data_ptr(), grads[0].defined() ? pointer<void>(grads[0]) : nullptr,
                                                            grads[1].defined() ? pointer<void>(grads[1]) : nullptr, &Scratch::alloc, &scratch,
                                                            current_stream(device)));
        }
        return first_order_only_in_inputs(std::move(grads), upstream[0]);
    }
};

Tensor linear_cross_entropy(const Tensor& features, const Tensor& table, const Tensor& targets, double scale, const std::string& reduction) {
    TORCH_CHECK_VALUE(table.dim() == 2, "efgs: the table must have two dimensions, got ", table.dim());
    TORCH_CHECK_VALUE(features.dim() >= 1 && features.size(-1) == table.size(1), "efgs: features must have the table's ", table.size(1),
                      " columns, got ", features.sizes());
    TORCH_CHECK_VALUE(targets.sizes() == features.sizes().slice(0, features.dim() - 1), "efgs: targets must have the features' shape without its columns, ",
                      features.sizes(), ", got ", targets.sizes());
    check_index_type("targets", targets);
    element_type("the table", table.scalar_type());
    TORCH_CHECK_VALUE(features.scalar_type() == table.scalar_type(), "efgs: features must have the table's type, ", table.dtype(), ", got ", features.dtype());
    check_dense("the table", table, table.device());
    check_dense("features", features, table.device());
    check_dense("targets", targets, table.device());
    TORCH_CHECK_VALUE(std::isfinite(scale) && std::isfinite(static_cast<float>(scale)), "efgs: the cross entropy's scale must be finite");
    check_no_tangent("linear_cross_entropy", features);
    check_no_tangent("linear_cross_entropy", table);
    EntropyCall c;
    if (reduction == "none") c.reduction = EFGS_EACH;
    else if (reduction == "sum") c.reduction = EFGS_SUM;
    else TORCH_CHECK_VALUE(reduction == "mean", "efgs: reduction must be none, sum or mean, got ", reduction);
    const c10::DeviceGuard guard(table.device());
    c.scale = scale;
    c.n = targets.numel();
    c.targets = targets.detach().contiguous();
    c.features = rows_of(features.detach().reshape({c.n, table.size(1)}));
    if (!needs_graph(features) && !needs_graph(table)) return entropy_forward(c, table.detach(), nullptr);
    return LinearCrossEntropy::apply(features, table, c);
}

// ---- dropout -----------------------------------------------------------------------------------------------------------

struct DropoutCall {
    double p = 0.0;
    uint64_t seed = 0, offset = 0;
    Tensor seed_at;   // or undefined
};

Tensor dropped(const Tensor& x, const Tensor& residual, const DropoutCall& c) {
    const Tensor from = x.contiguous(), beside = residual.defined() ? residual.contiguous() : residual;
    const Tensor out = at::empty(x.sizes(), x.options().requires_grad(false).memory_format(at::MemoryFormat::Contiguous));
    check_status(efgs_dropout(pointer<void>(from), beside.defined() ? pointer<void>(beside) : nullptr, pointer<void>(out), x.numel(),
                              element_type("dropout's input", x.scalar_type()), c.p, c.seed,
                              c.seed_at.defined() ? pointer<uint64_t>(c.seed_at) : nullptr, c.offset, current_stream(x.device())));
    return out;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& residual, const DropoutCall& c) {
        ctx->saved_data["p"] = c.p;
        ctx->saved_data["seed"] = static_cast<int64_t>(c.seed);
        ctx->saved_data["offset"] = static_cast<int64_t>(c.offset);
        ctx->saved_data["type"] = x.scalar_type();
        ctx->saved_data["residual"] = residual.has_value();
        if (c.seed_at.defined()) ctx->save_for_backward({c.seed_at});
        return dropped(x.detach(), residual ? residual->detach() : Tensor(), c);
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list grads(3);
        {
            at::NoGradGuard no_grad;
            DropoutCall c;
            c.p = ctx->saved_data["p"].toDouble();
            c.seed = static_cast<uint64_t>(ctx->saved_data["seed"].toInt());
            c.offset = static_cast<uint64_t>(ctx->saved_data["offset"].toInt());
            if (!saved.empty()) c.seed_at = saved[0];
            const Tensor& g = upstream[0];
            TORCH_CHECK_VALUE(g.device().is_cuda() && g.scalar_type() == ctx->saved_data["type"].toScalarType() &&
                                  (!c.seed_at.defined() || (c.seed_at.device() == g.device() && c.seed_at.scalar_type() == at::kLong && c.seed_at.numel() == 1)),
                              "efgs: dropout's gradient must have the output's type, on its device");
            const c10::DeviceGuard guard(g.device());
            if (ctx->needs_input_grad(0)) grads[0] = dropped(g.detach(), Tensor(), c);
            // (the upstream itself: a leaf takes a gradient that nobody else holds as its own, and a detached one would pass for such)
            if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) grads[1] = g;
        }
        return first_order_only(std::move(grads), upstream[0]);
    }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, const c10::optional<Tensor>& seed_at, uint64_t offset, const c10::optional<Tensor>& residual) {
    const at::Device device = x.device();
    check_dense("dropout's input", x, device);
    element_type("dropout's input", x.scalar_type());
    TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "efgs: the dropout probability must lie in [0, 1], got ", p);
    check_no_tangent("dropout", x);
    DropoutCall c;
    c.p = p;
    c.seed = seed;
    c.offset = offset;
    if (seed_at) {
        check_dense("dropout's seed", *seed_at, device);
        TORCH_CHECK_VALUE(seed_at->scalar_type() == at::kLong && seed_at->numel() == 1, "efgs: dropout's seed must be one int64 value, got ",
                          seed_at->dtype(), " of shape ", seed_at->sizes());
        c.seed_at = *seed_at;
    }
    Tensor beside;
    if (residual) {
        beside = *residual;
        check_dense("dropout's residual", beside, device);
        TORCH_CHECK_VALUE(beside.sizes() == x.sizes() && beside.scalar_type() == x.scalar_type(), "efgs: dropout's residual must have its input's shape and type, ",
                          x.sizes(), " ", x.dtype(), ", got ", beside.sizes(), " ", beside.dtype());
        check_no_tangent("dropout", beside);
    }
    const c10::DeviceGuard guard(device);
    if (!needs_graph(x) && !needs_graph(beside)) return dropped(x.detach(), beside.defined() ? beside.detach() : beside, c);
    return Dropout::apply(x, residual, c);
}

// (seed, offset) of a torch generator for the draws of one call, which moves it on by four, as one step under its lock: what other threads draw meanwhile
// has other offsets
std::pair<uint64_t, uint64_t> draw_counters(at::Generator generator) {
    const std::lock_guard<std::mutex> lock(generator.mutex());
    const uint64_t seed = generator.current_seed(), offset = generator.get_offset();
    generator.set_offset(offset + 4);
    return {seed, offset};
}

// ---- balance loss ------------------------------------------------------------------------------------------------------

struct BalanceCall {
    Tensor logits, indices;   // contiguous
    int64_t n = 0, experts = 0, chosen = 0;
    int32_t type = 0;
};

struct BalanceResult {
    Tensor loss, counts, share;
};

BalanceResult balance_forward(const BalanceCall& c) {
    const at::Device device = c.logits.device();
    const auto options = at::TensorOptions().device(device);
    BalanceResult r{at::empty({}, options.dtype(at::kFloat)), at::empty({c.experts}, options.dtype(at::kLong)),
                    at::empty({c.experts + 1}, options.dtype(at::kFloat))};
    Scratch scratch(device);
    check_status(efgs_balance_loss_forward(pointer<void>(c.logits), pointer<void>(c.indices), static_cast<int>(c.indices.element_size()), c.n, c.experts,
                                           c.chosen, c.type, pointer<float>(r.loss), pointer<int64_t>(r.counts), pointer<float>(r.share), &Scratch::alloc,
                                           &scratch, current_stream(device)));
    return r;
}

struct BalanceLoss : torch::autograd::Function<BalanceLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const BalanceCall& c) {
        const BalanceResult r = balance_forward(c);
        ctx->saved_data["chosen"] = c.chosen;
        ctx->save_for_backward({logits, c.indices, r.share});
        ctx->mark_non_differentiable({r.counts});
        return {r.loss, r.counts};
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list grads(2);
        {
            at::NoGradGuard no_grad;
            const Tensor logits = saved[0].detach().contiguous(), indices = saved[1].contiguous(), share = saved[2].contiguous();
            const at::Device device = logits.device();
            const int64_t experts = logits.size(-1), n = logits.numel() / experts, chosen = ctx->saved_data["chosen"].toInt();
            TORCH_CHECK_VALUE(indices.device() == device && indices.numel() == n * chosen && share.device() == device && share.numel() == experts + 1 &&
                                  share.scalar_type() == at::kFloat && (indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong),
                              "efgs: the balance loss's saved tensors are not what its forward saved");
            const c10::DeviceGuard guard(device);
            const Tensor g = float_upstream(upstream[0], 1, device);
            grads[0] = at::empty(logits.sizes(), logits.options());
            check_status(efgs_balance_loss_backward(pointer<void>(logits), pointer<void>(indices), static_cast<int>(indices.element_size()), n, experts, chosen,
                                                    element_type("logits", logits.scalar_type()), pointer<float>(share), pointer<float>(g),
                                                    pointer<void>(grads[0]), current_stream(device)));
        }
        return first_order_only_in_inputs(std::move(grads), upstream[0]);
    }
};

std::pair<Tensor, Tensor> balance_loss(const Tensor& logits, const Tensor& indices) {
    TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1, "efgs: logits must have a last dimension of experts, got ", logits.sizes());
    const at::IntArrayRef rows = logits.sizes().slice(0, logits.dim() - 1);
    const bool one = indices.sizes() == rows, several = indices.dim() == logits.dim() && indices.sizes().slice(0, logits.dim() - 1) == rows;
    TORCH_CHECK_VALUE(one || several, "efgs: indices must have the logits' shape without its experts, or with choices in their place, ", logits.sizes(),
                      ", got ", indices.sizes());
    check_index_type("indices", indices);
    check_dense("logits", logits, logits.device());
    check_dense("indices", indices, logits.device());
    check_no_tangent("balance_loss", logits);
    BalanceCall c;
    c.type = element_type("logits", logits.scalar_type());
    c.experts = logits.size(-1);
    c.n = logits.numel() / c.experts;
    c.chosen = one ? 1 : indices.size(-1);
    const c10::DeviceGuard guard(logits.device());
    c.logits = logits.detach().contiguous();
    c.indices = indices.detach().contiguous();
    if (!needs_graph(logits)) {
        const BalanceResult r = balance_forward(c);
        return {r.loss, r.counts};
    }
    const variable_list out = BalanceLoss::apply(logits, c);
    return {out[0], out[1]};
}

}  // namespace

void register_losses(py::module_& m) {
    m.def("linear_cross_entropy", torch::wrap_pybind_function_no_gil(linear_cross_entropy));
    m.def("dropout", torch::wrap_pybind_function_no_gil(dropout));
    m.def("draw_counters", torch::wrap_pybind_function_no_gil(draw_counters));
    m.def("balance_loss", torch::wrap_pybind_function_no_gil(balance_loss));
}

}  // namespace efgs_torch
