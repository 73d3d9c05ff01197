// The training operators beside the rasterizer for Python: rows of a table by index as a C++ autograd function, the AdamW
// step over all tensors of an optimizer (gathered from its groups and states here: a step over many small tensors is bound
// by the host), the moments of 8-bit states and the gradient norm.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <string>

#include "torch_common.h"

namespace py = pybind11;

namespace efgs_torch {

namespace {

// ---- rows of a table by index ------------------------------------------------------------------------------------------

struct Rows {
    Tensor indices, table;
    int64_t n = 0, rows = 0, columns = 0;
    int32_t type = 0;
    double scale = 1.0;
    int64_t padding = -1;
};

Tensor lookup(const Rows& r) {
    std::vector<int64_t> shape = r.indices.sizes().vec();
    shape.push_back(r.columns);
    const Tensor out = at::empty(shape, r.table.options().requires_grad(false));
    check_status(efgs_embedding_forward(r.n > 0 ? r.indices.data_ptr() : nullptr, static_cast<int>(r.indices.element_size()), r.n,
                                        r.table.numel() > 0 ? r.table.data_ptr() : nullptr, r.rows, r.columns, r.rows > 1 ? r.table.stride(0) : r.columns,
                                        r.type, static_cast<float>(r.scale), out.numel() > 0 ? out.data_ptr() : nullptr,
                                        current_stream(r.table.device())));
    return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& table, const Rows& r) {
        ctx->saved_data["rows"] = r.rows;
        ctx->saved_data["columns"] = r.columns;
        ctx->saved_data["scale"] = r.scale;
        ctx->saved_data["padding"] = r.padding;
        ctx->save_for_backward({r.indices});
        (void)table;
        return lookup(r);
    }

    static variable_list backward(AutogradContext* ctx, variable_list upstream) {
        const variable_list saved = ctx->get_saved_variables();
        variable_list grads;
        {
            at::NoGradGuard no_grad;
            grads = {gradient(ctx, saved[0], upstream[0]), Tensor()};
        }
        return first_order_only(std::move(grads), upstream[0]);
    }

    static Tensor gradient(AutogradContext* ctx, const Tensor& saved, const Tensor& upstream) {
        const int64_t rows = ctx->saved_data["rows"].toInt(), columns = ctx->saved_data["columns"].toInt();
        // (a node called directly is given whatever its caller has, and hooks on saved tensors return what they like)
        const at::Device device = upstream.device();
        TORCH_CHECK_VALUE(device.is_cuda() && saved.device() == device && (saved.scalar_type() == at::kInt || saved.scalar_type() == at::kLong),
                          "efgs: the embedding's indices must be int32 or int64 on the gradient's device, got ", saved.dtype(), " on ", saved.device());
        const at::IntArrayRef sizes = upstream.sizes();
        TORCH_CHECK_VALUE(!sizes.empty() && sizes.back() == columns && sizes.slice(0, sizes.size() - 1) == saved.sizes(),
                          "efgs: the embedding's gradient must have the output's shape, the indices' ", saved.sizes(), " and ", columns, " columns, got ", sizes);
        const c10::DeviceGuard guard(device);
        const Tensor indices = saved.contiguous(), grad_out = upstream.contiguous();
        const Tensor out = at::empty({rows, columns}, grad_out.options());
        Scratch scratch(device);
        check_status(efgs_embedding_backward(indices.numel() > 0 ? indices.data_ptr() : nullptr, static_cast<int>(indices.element_size()),
                                             indices.numel(), grad_out.numel() > 0 ? grad_out.data_ptr() : nullptr, rows, columns,
                                             element_type("the gradient", grad_out.scalar_type()), static_cast<float>(ctx->saved_data["scale"].toDouble()),
                                             ctx->saved_data["padding"].toInt(), out.numel() > 0 ? out.data_ptr() : nullptr, &Scratch::alloc, &scratch,
                                             current_stream(device)));
        return out;
    }
};

Tensor embedding(const Tensor& indices, const Tensor& table, double scale, const c10::optional<int64_t>& padding_idx) {
    TORCH_CHECK_VALUE(table.dim() == 2, "efgs: the table must have two dimensions, got ", table.dim());
    TORCH_CHECK_VALUE(indices.scalar_type() == at::kInt || indices.scalar_type() == at::kLong, "efgs: indices must be int32 or int64, got ",
                      indices.dtype());
    TORCH_CHECK_VALUE(table.device().is_cuda(), "efgs: the table must be on a GPU device, got ", table.device());
    TORCH_CHECK_VALUE(indices.device() == table.device(), "efgs: indices are on ", indices.device(), ", expected ", table.device());
    TORCH_CHECK_VALUE(std::isfinite(scale), "efgs: the embedding scale must be finite");
    // (a lookup that needs no graph passes the autograd function by, which would refuse: its result would have lost the tangent)
    TORCH_CHECK_NOT_IMPLEMENTED(!table._fw_grad(/*level=*/0).defined(), "efgs: embedding has no forward-mode derivative");
    Rows r;
    r.type = element_type("the table", table.scalar_type());
    r.rows = table.size(0);
    r.columns = table.size(1);
    r.scale = scale;
    if (padding_idx.has_value()) {
        TORCH_CHECK_VALUE(*padding_idx >= -r.rows && *padding_idx < r.rows, "efgs: padding_idx must lie within the table's ", r.rows, " rows, got ",
                          *padding_idx);
        r.padding = *padding_idx < 0 ? *padding_idx + r.rows : *padding_idx;
    }
    const c10::DeviceGuard guard(table.device());
    r.indices = indices.detach().contiguous();
    r.n = r.indices.numel();
    r.table = table.detach();
    if (r.columns > 1 && r.table.stride(1) != 1) r.table = r.table.contiguous();
    if (!(at::GradMode::is_enabled() && table.requires_grad())) return lookup(r);
    return Embedding::apply(table, r);
}

// ---- gradient norm -----------------------------------------------------------------------------------------------------

Tensor norm_of(const std::vector<efgs_norm_tensor>& tensors, at::Device device) {
    const c10::DeviceGuard guard(device);
    const Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(device));
    Scratch scratch(device);
    check_status(efgs_grad_norm(tensors.data(), static_cast<int64_t>(tensors.size()), static_cast<float*>(norm.data_ptr()), &Scratch::alloc, &scratch,
                                current_stream(device)));
    return norm;
}

Tensor grad_norm(const std::vector<Tensor>& tensors) {
    TORCH_CHECK_VALUE(!tensors.empty(), "efgs: grad_norm needs at least one tensor");
    const at::Device device = tensors[0].device();
    TORCH_CHECK_VALUE(device.is_cuda(), "efgs: grad_norm runs on a GPU device, got ", device);
    std::vector<Tensor> kept;
    std::vector<efgs_norm_tensor> native;
    for (const Tensor& t : tensors) {
        TORCH_CHECK_VALUE(t.device() == device, "efgs: grad_norm's tensors must live on one device");
        TORCH_CHECK_VALUE(t.layout() == at::kStrided, "efgs: grad_norm's tensors must be dense");
        const int32_t type = element_type("a gradient", t.scalar_type());
        if (t.numel() == 0) continue;
        const c10::DeviceGuard guard(device);
        kept.push_back(t.detach().contiguous());
        native.push_back({kept.back().data_ptr(), t.numel(), type, 0});
    }
    return norm_of(native, device);
}

// ---- AdamW -------------------------------------------------------------------------------------------------------------

// names of the state's entries, kept for the interpreter's life
PyObject* name(int k) {
    static PyObject* const names[] = {PyUnicode_InternFromString("step"),           PyUnicode_InternFromString("exp_avg"),
                                      PyUnicode_InternFromString("exp_avg_sq"),     PyUnicode_InternFromString("exp_avg_ratio"),
                                      PyUnicode_InternFromString("exp_avg_sq_root"), PyUnicode_InternFromString("root_scale"),
                                      PyUnicode_InternFromString("ratio_bound")};
    return names[k];
}
enum { step_name, exp_avg_name, exp_avg_sq_name, ratio_name, root_name, scale_name, bound_name };

void set_entry(PyObject* dict, int key, PyObject* value) {  // takes `value` over
    if (!value) throw py::error_already_set();
    const int rc = PyDict_SetItem(dict, name(key), value);
    Py_DECREF(value);
    if (rc != 0) throw py::error_already_set();
}

const Tensor& tensor_entry(PyObject* dict, int key, const Tensor& param, at::ScalarType type, int64_t numel) {
    PyObject* const item = PyDict_GetItemWithError(dict, name(key));
    TORCH_CHECK_VALUE(item && THPVariable_Check(item), "efgs: AdamW: a parameter's state lacks ", PyUnicode_AsUTF8(name(key)),
                      " (state_bits differs from the state's?)");
    const Tensor& t = THPVariable_Unpack(item);
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.numel() == numel && t.is_contiguous() && t.device() == param.device(), "efgs: AdamW: state entry ",
                      PyUnicode_AsUTF8(name(key)), " must hold ", numel, " contiguous values of ", type, " on ", param.device());
    return t;
}

double bound_entry(PyObject* dict) {
    PyObject* const item = PyDict_GetItemWithError(dict, name(bound_name));
    TORCH_CHECK_VALUE(item && PyFloat_Check(item), "efgs: AdamW: a parameter's 8-bit state lacks its ratio_bound");
    return PyFloat_AsDouble(item);
}

int64_t step_entry(PyObject* dict) {
    PyObject* const item = PyDict_GetItemWithError(dict, name(step_name));
    TORCH_CHECK_VALUE(item && PyLong_Check(item), "efgs: AdamW: a parameter's state needs its step as an int");
    return PyLong_AsLongLong(item);
}

int64_t blocks_of(int64_t n) { return (n + 255) / 256; }

// the state of a parameter, made of zeros where there is none yet
PyObject* state_of(PyObject* states, PyObject* key, const Tensor& param, int bits, double bound) {
    PyObject* state = PyDict_GetItemWithError(states, key);
    if (!state) {
        if (PyErr_Occurred()) throw py::error_already_set();
        const py::dict made;
        if (PyDict_SetItem(states, key, made.ptr()) != 0) throw py::error_already_set();
        state = made.ptr();  // (held by `states`)
    }
    TORCH_CHECK_VALUE(PyDict_Check(state), "efgs: AdamW: a parameter's state must be a dict");
    if (PyDict_GET_SIZE(state) > 0) return state;
    const c10::DeviceGuard guard(param.device());
    const auto options = at::TensorOptions().device(param.device());
    // (all of them made before the first is kept: memory may run out)
    const auto type = options.dtype(bits == 32 ? at::kFloat : at::kByte);
    const Tensor first = at::zeros(param.sizes(), type), second = at::zeros(param.sizes(), type);
    if (bits == 32) {
        set_entry(state, exp_avg_name, THPVariable_Wrap(first));
        set_entry(state, exp_avg_sq_name, THPVariable_Wrap(second));
    } else {
        const Tensor scale = at::zeros({blocks_of(param.numel())}, options.dtype(at::kFloat));
        set_entry(state, ratio_name, THPVariable_Wrap(first));
        set_entry(state, root_name, THPVariable_Wrap(second));
        set_entry(state, scale_name, THPVariable_Wrap(scale));
        set_entry(state, bound_name, PyFloat_FromDouble(bound));
    }
    set_entry(state, step_name, PyLong_FromLongLong(0));
    return state;
}

PyObject* group_entry(PyObject* group, PyObject* key) {
    PyObject* const item = PyDict_GetItemWithError(group, key);
    TORCH_CHECK_VALUE(item, "efgs: AdamW: a parameter group lacks ", PyUnicode_AsUTF8(key));
    return item;
}

double as_double(PyObject* item) {
    const double x = PyFloat_AsDouble(item);  // (numbers, and whatever turns into a float: a tensor of one value)
    if (x == -1.0 && PyErr_Occurred()) throw py::error_already_set();
    return x;
}

efgs_adamw_group native_group(PyObject* group) {
    static PyObject* const lr_name = PyUnicode_InternFromString("lr");
    static PyObject* const betas_name = PyUnicode_InternFromString("betas");
    static PyObject* const eps_name = PyUnicode_InternFromString("eps");
    static PyObject* const decay_name = PyUnicode_InternFromString("weight_decay");
    static PyObject* const bits_name = PyUnicode_InternFromString("state_bits");
    efgs_adamw_group native{};
    PyObject* const lr = group_entry(group, lr_name);
    if (PyList_Check(lr) || PyTuple_Check(lr)) {
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(lr);
        TORCH_CHECK_VALUE(n >= 1 && n <= 7, "efgs: between 1 and 7 learning rates are supported");
        for (Py_ssize_t k = 0; k < n; k++) native.lrs[k] = as_double(PySequence_Fast_GET_ITEM(lr, k));
        native.n_lrs = static_cast<int32_t>(n);
    } else {
        native.lrs[0] = as_double(lr);
        native.n_lrs = 1;
    }
    PyObject* const betas = group_entry(group, betas_name);
    TORCH_CHECK_VALUE((PyTuple_Check(betas) || PyList_Check(betas)) && PySequence_Fast_GET_SIZE(betas) == 2, "efgs: AdamW: betas must be two numbers");
    native.beta1 = as_double(PySequence_Fast_GET_ITEM(betas, 0));
    native.beta2 = as_double(PySequence_Fast_GET_ITEM(betas, 1));
    native.eps = as_double(group_entry(group, eps_name));
    native.weight_decay = as_double(group_entry(group, decay_name));
    native.state_bits = static_cast<int32_t>(as_double(group_entry(group, bits_name)));
    return native;
}

// One step over every parameter that has a gradient. groups: the optimizer's param_groups; states: its state. Returns the gradients' norm where it clips. Nothing has changed if this throws
// before the launch (states of zeros may have been made).
c10::optional<Tensor> adamw_step(const py::list& groups, const py::dict& states, const c10::optional<double>& max_grad_norm, uint32_t seed) {
    at::NoGradGuard no_grad;
    struct Entry {
        Tensor param;
        PyObject* state;
        int64_t step;
        double bound;  // to be written, 0: none
    };
    std::vector<Entry> entries;
    std::vector<Tensor> kept;
    std::vector<efgs_adamw_tensor> tensors;
    std::vector<efgs_norm_tensor> norms;
    std::vector<efgs_adamw_group> native_groups;
    c10::optional<at::Device> device;
    for (const py::handle item : groups) {
        TORCH_CHECK_VALUE(PyDict_Check(item.ptr()), "efgs: AdamW: a parameter group must be a dict");
        native_groups.push_back(native_group(item.ptr()));
    }
    // (a step over no tensors: the groups' values are checked before states are made by them)
    check_status(efgs_adamw_step(nullptr, 0, native_groups.data(), static_cast<int>(native_groups.size()), nullptr, 0.0, seed, nullptr));
    int32_t group = -1;
    for (const py::handle item : groups) {
        static PyObject* const params_name = PyUnicode_InternFromString("params");
        PyObject* const params = group_entry(item.ptr(), params_name);
        TORCH_CHECK_VALUE(PyList_Check(params), "efgs: AdamW: a group's parameters must be a list");
        const size_t most = tensors.size() + static_cast<size_t>(PyList_GET_SIZE(params));
        entries.reserve(most);
        tensors.reserve(most);
        norms.reserve(max_grad_norm ? most : 0);
        const efgs_adamw_group& native = native_groups[static_cast<size_t>(++group)];
        const int bits = native.state_bits;
        const double bound = bits == 8 ? efgs_adamw_ratio_bound(native.beta1, native.beta2) : 0.0;
        for (Py_ssize_t k = 0; k < PyList_GET_SIZE(params); k++) {
            PyObject* const key = PyList_GET_ITEM(params, k);
            TORCH_CHECK_VALUE(THPVariable_Check(key), "efgs: AdamW: parameters must be tensors");
            const Tensor& param = THPVariable_Unpack(key);
            const Tensor& given = param.grad();
            if (!given.defined() || param.numel() == 0) continue;
            TORCH_CHECK_VALUE(param.device().is_cuda() && param.is_contiguous(), "efgs: AdamW: parameters must be contiguous GPU tensors");
            TORCH_CHECK_VALUE(!device || param.device() == *device, "efgs: AdamW: all parameters must live on one device");
            TORCH_CHECK_VALUE(given.layout() == at::kStrided && given.sizes() == param.sizes() && given.device() == param.device(),
                              "efgs: AdamW: a gradient must be a dense tensor of its parameter's shape and device");
            device = param.device();
            efgs_adamw_tensor t{};
            t.param_type = element_type("AdamW: a parameter", param.scalar_type());
            t.grad_type = element_type("AdamW: a gradient", given.scalar_type());
            if (given.is_contiguous()) {
                t.grad = given.data_ptr();
            } else {
                const c10::DeviceGuard guard(*device);
                kept.push_back(given.contiguous());
                t.grad = kept.back().data_ptr();
            }
            PyObject* const state = state_of(states.ptr(), key, param, bits, bound);
            const int64_t n = param.numel();
            double written = 0.0;
            if (bits == 32) {
                t.exp_avg = tensor_entry(state, exp_avg_name, param, at::kFloat, n).data_ptr();
                t.exp_avg_sq = tensor_entry(state, exp_avg_sq_name, param, at::kFloat, n).data_ptr();
            } else {
                t.exp_avg = tensor_entry(state, ratio_name, param, at::kByte, n).data_ptr();
                t.exp_avg_sq = tensor_entry(state, root_name, param, at::kByte, n).data_ptr();
                t.root_scale = static_cast<float*>(tensor_entry(state, scale_name, param, at::kFloat, blocks_of(n)).data_ptr());
                t.ratio_bound = bound_entry(state);
                if (t.ratio_bound != bound) written = bound;
            }
            t.param = param.data_ptr();
            t.n_elements = n;
            t.step = step_entry(state) + 1;
            t.group = group;
            if (max_grad_norm) norms.push_back({t.grad, n, t.grad_type, 0});
            tensors.push_back(t);
            entries.push_back({param, state, t.step, written});
        }
    }
    if (entries.empty()) return c10::nullopt;
    const c10::DeviceGuard guard(*device);
    TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None,
                "efgs: AdamW counts its steps on the host and cannot be captured into a graph");
    c10::optional<Tensor> norm;
    if (max_grad_norm) norm = norm_of(norms, *device);
    check_status(efgs_adamw_step(tensors.data(), static_cast<int64_t>(tensors.size()), native_groups.data(), static_cast<int>(native_groups.size()),
                                 norm ? static_cast<const float*>(norm->data_ptr()) : nullptr, max_grad_norm.value_or(0.0), seed,
                                 current_stream(*device)));
    for (const Entry& e : entries) {
        e.param.unsafeGetTensorImpl()->bump_version();
        set_entry(e.state, step_name, PyLong_FromLongLong(e.step));
        if (e.bound != 0.0) set_entry(e.state, bound_name, PyFloat_FromDouble(e.bound));
    }
    return norm;
}

// (exp_avg, exp_avg_sq) of every parameter; 32-bit states as they are, 8-bit ones as new tensors
std::vector<std::pair<Tensor, Tensor>> adamw_moments(const py::list& params, const py::dict& states) {
    std::vector<std::pair<Tensor, Tensor>> out;
    std::vector<efgs_adamw_state> native;
    c10::optional<at::Device> device;
    for (const py::handle item : params) {
        PyObject* const key = item.ptr();
        TORCH_CHECK_VALUE(THPVariable_Check(key), "efgs: AdamW: parameters must be tensors");
        const Tensor& param = THPVariable_Unpack(key);
        PyObject* const state = PyDict_GetItemWithError(states.ptr(), key);
        TORCH_CHECK_VALUE(state && PyDict_Check(state) && PyDict_GET_SIZE(state) > 0, "efgs: AdamW: a parameter has no state yet");
        const int64_t n = param.numel();
        if (PyDict_GetItemWithError(state, name(exp_avg_name))) {
            out.emplace_back(tensor_entry(state, exp_avg_name, param, at::kFloat, n), tensor_entry(state, exp_avg_sq_name, param, at::kFloat, n));
            continue;
        }
        TORCH_CHECK_VALUE(param.device().is_cuda(), "efgs: AdamW: 8-bit states are read on a GPU device, got ", param.device());
        TORCH_CHECK_VALUE(!device || param.device() == *device, "efgs: AdamW: all parameters must live on one device");
        device = param.device();
        const auto options = at::TensorOptions().dtype(at::kFloat).device(param.device());
        out.emplace_back(at::empty(param.sizes(), options), at::empty(param.sizes(), options));
        efgs_adamw_state s{};
        s.ratios = static_cast<const uint8_t*>(tensor_entry(state, ratio_name, param, at::kByte, n).data_ptr());
        s.roots = static_cast<const uint8_t*>(tensor_entry(state, root_name, param, at::kByte, n).data_ptr());
        s.root_scale = static_cast<const float*>(tensor_entry(state, scale_name, param, at::kFloat, blocks_of(n)).data_ptr());
        s.exp_avg = static_cast<float*>(out.back().first.data_ptr());
        s.exp_avg_sq = static_cast<float*>(out.back().second.data_ptr());
        s.ratio_bound = bound_entry(state);
        s.n_elements = n;
        native.push_back(s);
    }
    if (!native.empty()) {
        const c10::DeviceGuard guard(*device);
        check_status(efgs_adamw_moments(native.data(), static_cast<int64_t>(native.size()), current_stream(*device)));
    }
    return out;
}

}  // namespace

void register_training(py::module_& m) {
    m.def("embedding", torch::wrap_pybind_function_no_gil(embedding));
    m.def("grad_norm", torch::wrap_pybind_function_no_gil(grad_norm));
    // (these read the optimizer's Python objects and keep the interpreter's lock)
    m.def("adamw_step", torch::wrap_pybind_function(adamw_step));
    m.def("adamw_moments", torch::wrap_pybind_function(adamw_moments));
}

}  // namespace efgs_torch
