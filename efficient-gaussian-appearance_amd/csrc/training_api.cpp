// C entry points of the training operators beside the rasterizer: AdamW over many tensors with 32-bit and 8-bit states,
// the gradient norm, and rows of a table by index with their gradient (include/efgs.h). Arguments are checked here, before
// any device work; nothing thrown leaves an entry point.
#include <cmath>
#include <exception>
#include <vector>

#include "../../include/efgs.h"
#include "internal.h"

using namespace efgs;

namespace {

int fail(int code, const std::string& msg) {
    set_error(msg);
    return code;
}

template <typename F>
int guarded(F&& f) {
    try {
        return f();
    } catch (const std::exception& e) {
        return fail(EFGS_ERR_ALLOC, std::string("host failure: ") + e.what());
    } catch (...) {
        return fail(EFGS_ERR_ALLOC, "host failure");
    }
}

bool known_type(int32_t type) { return type == EFGS_FLOAT || type == EFGS_BFLOAT16 || type == EFGS_HALF; }

// the fault of a group's values, or null
const char* group_fault(const efgs_adamw_group& g) {
    if (g.n_lrs < 1 || g.n_lrs > adam_max_lrs) return "between 1 and 7 learning rates are supported";
    for (int k = 0; k < g.n_lrs; k++)
        if (!std::isfinite(g.lrs[k])) return "adamw learning rates must be finite";
    if (!(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0)) return "adamw betas must lie in [0, 1)";
    if (!(g.eps >= 0.0 && std::isfinite(g.eps))) return "adamw eps must be finite and not negative";
    if (!std::isfinite(g.weight_decay)) return "adamw weight decay must be finite";
    if (g.state_bits != 32 && g.state_bits != 8) return "adamw states have 32 or 8 bits";
    if (g.state_bits == 8 && !(g.beta1 * g.beta1 < g.beta2)) return "8-bit adamw states need beta1^2 < beta2";
    return nullptr;
}

AdamWGroupDevice device_group(const efgs_adamw_group& g, int64_t step, double ratio_bound, uint32_t seed) {
    AdamWGroupDevice d{};
    // An eps below the normal floats has no reciprocal in the hardware (0 times it would be no number for zero moments): the quotient's
    // denominator is held times 2^32 then, and at least the least float, and so is the rate.
    const bool tiny = g.eps > 0.0 && g.eps < 0x1p-126;
    const double eps = tiny ? std::fmax(g.eps, 0x1p-149) : g.eps, factor = tiny ? 0x1p32 : 1.0;
    const double step_factor = factor / (1.0 - std::pow(g.beta1, static_cast<double>(step)));
    for (int k = 0; k < g.n_lrs; k++) {
        d.rates[k] = static_cast<float>(g.lrs[k] * step_factor);
        d.decays[k] = static_cast<float>(1.0 - g.lrs[k] * g.weight_decay);
    }
    d.n_lrs = static_cast<uint32_t>(g.n_lrs);
    d.beta1 = static_cast<float>(g.beta1);
    d.beta1_rest = static_cast<float>(1.0 - g.beta1);
    d.beta2 = static_cast<float>(g.beta2);
    d.beta2_rest = static_cast<float>(1.0 - g.beta2);
    d.eps = static_cast<float>(eps * factor);
    d.root_factor = static_cast<float>(factor / std::sqrt(1.0 - std::pow(g.beta2, static_cast<double>(step))));
    if (g.state_bits == 8) {
        d.ratio_encode = static_cast<float>(adamw_ratio_top / efgs_adamw_ratio_bound(g.beta1, g.beta2));
        d.ratio_decode = static_cast<float>(ratio_bound / adamw_ratio_top);
        d.key = adamw_mix(adamw_mix(seed) + static_cast<uint32_t>(step));
    }
    return d;
}

// The groups that tensors of one step and, with 8 bits, one ratio bound share; most programs have one for each of theirs.
class SharedGroups {
  public:
    SharedGroups(const efgs_adamw_group* groups, int n_groups, uint32_t seed) : groups_(groups), seed_(seed), last_(static_cast<size_t>(n_groups), none) {}
    uint32_t of(int32_t group, int64_t step, double ratio_bound) {
        if (groups_[group].state_bits != 8) ratio_bound = 0.0;
        const uint32_t last = last_[static_cast<size_t>(group)];
        if (last != none && keys_[last].step == step && keys_[last].ratio_bound == ratio_bound) return last;
        uint32_t k = 0;
        while (k < keys_.size() && !(keys_[k].group == group && keys_[k].step == step && keys_[k].ratio_bound == ratio_bound)) k++;
        if (k == keys_.size()) {
            keys_.push_back({group, step, ratio_bound});
            device_.push_back(device_group(groups_[group], step, ratio_bound, seed_));
        }
        return last_[static_cast<size_t>(group)] = k;
    }
    const AdamWGroupDevice* data() const { return device_.data(); }

  private:
    static constexpr uint32_t none = 0xffffffffu;
    struct Key {
        int32_t group;
        int64_t step;
        double ratio_bound;
    };
    const efgs_adamw_group* groups_;
    uint32_t seed_;
    std::vector<uint32_t> last_;
    std::vector<Key> keys_;
    std::vector<AdamWGroupDevice> device_;
};

bool scale_pointer_ok(const void* p) { return p && reinterpret_cast<uintptr_t>(p) % alignof(float) == 0; }

EmbeddingArgs embedding_args(const void* indices, int index_bytes, int64_t n, int64_t rows, int64_t columns, int type, float scale) {
    EmbeddingArgs a{};
    a.indices = indices;
    a.index_bytes = index_bytes;
    a.type = type;
    a.n = static_cast<uint32_t>(n);
    a.rows = static_cast<uint32_t>(rows);
    a.columns = static_cast<uint32_t>(columns);
    a.scale = scale;
    return a;
}

const char* embedding_fault(const void* indices, int index_bytes, int64_t n, int64_t rows, int64_t columns, int type, float scale) {
    if (n < 0 || rows < 0 || columns < 0 || n > embedding_max || rows > embedding_max || columns > embedding_max)
        return "embedding sizes must lie between 0 and 2^31 - 1";
    if (index_bytes != 4 && index_bytes != 8) return "embedding indices have 4 or 8 bytes";
    if (!known_type(type)) return "unknown element type";
    if (!std::isfinite(scale)) return "the embedding scale must be finite";
    if (n > 0 && !indices) return "null embedding indices";
    return nullptr;
}

}  // namespace

extern "C" {

double efgs_adamw_ratio_bound(double beta1, double beta2) { return (1.0 - beta1) / std::sqrt((1.0 - beta2) * (1.0 - beta1 * beta1 / beta2)); }

int efgs_adamw_step(const efgs_adamw_tensor* tensors, int64_t n_tensors, const efgs_adamw_group* groups, int n_groups, const float* grad_norm,
                    double max_grad_norm, uint32_t seed, void* stream) {
    return guarded([&]() -> int {
        if (n_tensors < 0 || n_groups < 0 || (n_tensors > 0 && !tensors) || (n_groups > 0 && !groups))
            return fail(EFGS_ERR_INVALID_ARGUMENT, "invalid adamw tensors or groups");
        if (grad_norm && !(max_grad_norm > 0.0)) return fail(EFGS_ERR_INVALID_ARGUMENT, "the largest gradient norm must be positive");
        for (int g = 0; g < n_groups; g++)
            if (const char* fault = group_fault(groups[g])) return fail(EFGS_ERR_INVALID_ARGUMENT, fault);
        SharedGroups shared(groups, n_groups, seed);
        std::vector<AdamWTensor> wide;
        std::vector<AdamWTensor8> coded;
        std::vector<uint32_t> wide_groups, coded_groups;
        for (int64_t k = 0; k < n_tensors; k++) {
            const efgs_adamw_tensor& t = tensors[k];
            if (t.group < 0 || t.group >= n_groups) return fail(EFGS_ERR_INVALID_ARGUMENT, "adamw group out of range");
            if (t.n_elements < 0 || t.n_elements > adamw_max_elements) return fail(EFGS_ERR_INVALID_ARGUMENT, "adamw element count out of range");
            if (t.step < 1) return fail(EFGS_ERR_INVALID_ARGUMENT, "adamw step counts from 1");
            if (!known_type(t.param_type) || !known_type(t.grad_type)) return fail(EFGS_ERR_INVALID_ARGUMENT, "unknown element type");
            if (t.n_elements == 0) continue;
            if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return fail(EFGS_ERR_INVALID_ARGUMENT, "null adamw tensor");
            AdamWTensor8 d{};
            d.param = t.param;
            d.grad = t.grad;
            d.m = t.exp_avg;
            d.v = t.exp_avg_sq;
            d.set(static_cast<uint64_t>(t.n_elements), static_cast<uint32_t>(t.param_type), static_cast<uint32_t>(t.grad_type));
            if (groups[t.group].state_bits == 8) {
                if (!scale_pointer_ok(t.root_scale)) return fail(EFGS_ERR_INVALID_ARGUMENT, "8-bit adamw states need their block scales");
                if (!(t.ratio_bound > 0.0 && std::isfinite(t.ratio_bound))) return fail(EFGS_ERR_INVALID_ARGUMENT, "8-bit adamw states need their ratio bound");
                d.scale = t.root_scale;
                coded.push_back(d);
                coded_groups.push_back(shared.of(t.group, t.step, t.ratio_bound));
            } else {
                wide.push_back(d);
                wide_groups.push_back(shared.of(t.group, t.step, 0.0));
            }
        }
        hipStream_t s = static_cast<hipStream_t>(stream);
        const float max_norm = static_cast<float>(max_grad_norm);
        if (!launch_adamw(wide.data(), wide_groups.data(), wide.size(), shared.data(), grad_norm, max_norm, s)) return EFGS_ERR_HIP;
        if (!launch_adamw8(coded.data(), coded_groups.data(), coded.size(), shared.data(), grad_norm, max_norm, s)) return EFGS_ERR_HIP;
        return EFGS_OK;
    });
}

int efgs_adamw_moments(const efgs_adamw_state* states, int64_t n_states, void* stream) {
    return guarded([&]() -> int {
        if (n_states < 0 || (n_states > 0 && !states)) return fail(EFGS_ERR_INVALID_ARGUMENT, "invalid adamw states");
        std::vector<AdamWMomentsDevice> device;
        for (int64_t k = 0; k < n_states; k++) {
            const efgs_adamw_state& t = states[k];
            if (t.n_elements < 0 || t.n_elements > adamw_max_elements) return fail(EFGS_ERR_INVALID_ARGUMENT, "adamw element count out of range");
            if (t.n_elements == 0) continue;
            if (!t.ratios || !t.roots || !scale_pointer_ok(t.root_scale) || !t.exp_avg || !t.exp_avg_sq)
                return fail(EFGS_ERR_INVALID_ARGUMENT, "null adamw state");
            if (!(t.ratio_bound > 0.0 && std::isfinite(t.ratio_bound))) return fail(EFGS_ERR_INVALID_ARGUMENT, "8-bit adamw states need their ratio bound");
            AdamWMomentsDevice d{};
            d.ratios = t.ratios;
            d.roots = t.roots;
            d.scale = t.root_scale;
            d.m = t.exp_avg;
            d.v = t.exp_avg_sq;
            d.n = static_cast<uint64_t>(t.n_elements);
            d.ratio_decode = static_cast<float>(t.ratio_bound / adamw_ratio_top);
            device.push_back(d);
        }
        return launch_adamw_moments(device.data(), device.size(), static_cast<hipStream_t>(stream)) ? EFGS_OK : EFGS_ERR_HIP;
    });
}

int efgs_grad_norm(const efgs_norm_tensor* tensors, int64_t n_tensors, float* norm, efgs_alloc_fn alloc, void* alloc_ctx, void* stream) {
    return guarded([&]() -> int {
        if (n_tensors < 0 || (n_tensors > 0 && !tensors) || !norm || !alloc) return fail(EFGS_ERR_INVALID_ARGUMENT, "invalid gradient norm arguments");
        std::vector<NormTensorDevice> device;
        for (int64_t k = 0; k < n_tensors; k++) {
            const efgs_norm_tensor& t = tensors[k];
            if (t.n_elements < 0 || t.n_elements > adamw_max_elements) return fail(EFGS_ERR_INVALID_ARGUMENT, "gradient element count out of range");
            if (!known_type(t.type)) return fail(EFGS_ERR_INVALID_ARGUMENT, "unknown element type");
            if (t.n_elements == 0) continue;
            if (!t.data) return fail(EFGS_ERR_INVALID_ARGUMENT, "null gradient");
            device.push_back({t.data, static_cast<uint64_t>(t.n_elements) << 2 | static_cast<uint64_t>(t.type)});
        }
        const uint64_t partials = norm_partials(device.data(), device.size());
        if (partials > 0xffffffffull) return fail(EFGS_ERR_INVALID_ARGUMENT, "too many gradients");
        double* buffer = static_cast<double*>(alloc(alloc_ctx, static_cast<size_t>(partials > 0 ? partials : 1) * sizeof(double)));
        if (!buffer) return fail(EFGS_ERR_ALLOC, "allocation of the gradient norm's partial sums failed");
        return launch_grad_norm(device.data(), device.size(), buffer, norm, static_cast<hipStream_t>(stream)) ? EFGS_OK : EFGS_ERR_HIP;
    });
}

int efgs_embedding_forward(const void* indices, int index_bytes, int64_t n, const void* table, int64_t rows, int64_t columns, int64_t row_stride,
                           int type, float scale, void* out, void* stream) {
    return guarded([&]() -> int {
        if (const char* fault = embedding_fault(indices, index_bytes, n, rows, columns, type, scale)) return fail(EFGS_ERR_INVALID_ARGUMENT, fault);
        if (row_stride < 0) return fail(EFGS_ERR_INVALID_ARGUMENT, "negative row stride");
        if (n == 0 || columns == 0) return EFGS_OK;
        if (!out || (rows > 0 && !table)) return fail(EFGS_ERR_INVALID_ARGUMENT, "null embedding tensor");
        const EmbeddingArgs a = embedding_args(indices, index_bytes, n, rows, columns, type, scale);
        return launch_embedding_lookup(a, table, static_cast<uint64_t>(row_stride), out, static_cast<hipStream_t>(stream)) ? EFGS_OK : EFGS_ERR_HIP;
    });
}

int efgs_embedding_backward(const void* indices, int index_bytes, int64_t n, const void* grad_out, int64_t rows, int64_t columns, int type,
                            float scale, int64_t padding_row, void* grad_table, efgs_alloc_fn alloc, void* alloc_ctx, void* stream) {
    return guarded([&]() -> int {
        if (const char* fault = embedding_fault(indices, index_bytes, n, rows, columns, type, scale)) return fail(EFGS_ERR_INVALID_ARGUMENT, fault);
        if (rows == 0 || columns == 0) return EFGS_OK;
        if (!grad_table || (n > 0 && !grad_out) || !alloc) return fail(EFGS_ERR_INVALID_ARGUMENT, "null embedding tensor");
        const EmbeddingArgs a = embedding_args(indices, index_bytes, n, rows, columns, type, scale);
        if (!embedding_gradient_fits(a)) return fail(EFGS_ERR_INVALID_ARGUMENT, "too many embedding indices and rows");
        const uint32_t padding = padding_row >= 0 && padding_row < rows ? static_cast<uint32_t>(padding_row) : static_cast<uint32_t>(rows);
        void* workspace = alloc(alloc_ctx, embedding_gradient_bytes(a));
        if (!workspace) return fail(EFGS_ERR_ALLOC, "allocation of the embedding gradient's workspace failed");
        return launch_embedding_gradient(a, grad_out, padding, grad_table, workspace, static_cast<hipStream_t>(stream)) ? EFGS_OK : EFGS_ERR_HIP;
    });
}

}  // extern "C"
