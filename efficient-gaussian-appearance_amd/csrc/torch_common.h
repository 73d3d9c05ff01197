// What the Python extension's sources share: workspaces, status checks, streams, and gradients that have no second
// derivatives.
#pragma once
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include <map>
#include <mutex>
#include <utility>
#include <vector>

#include "../../include/efgs.h"

namespace efgs_torch {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// One device allocation per call, handed out by the library's bump allocator; requests beyond it get tensors of their
// own. The region follows the largest total requested so far (per call kind and device, with 1/16 headroom), so in
// steady state a call makes a single allocation.
class Workspace {
  public:
    enum Kind { forward = 0, backward = 1, decode = 2, forward_no_backward = 3 };

    Workspace(Kind kind, at::Device device) : key_(kind, device.index()), options_(at::TensorOptions().dtype(at::kByte).device(device)) {
        size_t capacity = 0;
        {
            std::lock_guard<std::mutex> lock(mutex());
            capacity = sizes()[key_];
        }
        tensors_.push_back(at::empty({static_cast<int64_t>(capacity > 256 ? capacity : 256)}, options_));
        ws_ = efgs_workspace{tensors_[0].data_ptr(), capacity, 0, 0, &Workspace::fallback, this};
    }
    Workspace(const Workspace&) = delete;
    Workspace& operator=(const Workspace&) = delete;

    efgs_workspace* context() { return &ws_; }

    // records the call's total for the next region; the tensors back every buffer that was handed out
    std::vector<Tensor> finish() {
        std::lock_guard<std::mutex> lock(mutex());
        size_t& size = sizes()[key_];
        if (ws_.requested > size) size = (ws_.requested + ws_.requested / 16 + 255) / 256 * 256;
        return std::move(tensors_);
    }

  private:
    static void* fallback(void* self, size_t bytes) noexcept {
        try {
            Workspace* w = static_cast<Workspace*>(self);
            w->tensors_.push_back(at::empty({static_cast<int64_t>(bytes > 0 ? bytes : 1)}, w->options_));
            return w->tensors_.back().data_ptr();
        } catch (...) {  // (out of memory: the library reports the failed allocation)
            return nullptr;
        }
    }
    static std::mutex& mutex() {
        static std::mutex m;
        return m;
    }
    static std::map<std::pair<int, int>, size_t>& sizes() {
        static std::map<std::pair<int, int>, size_t> s;
        return s;
    }

    std::pair<int, int> key_;
    at::TensorOptions options_;
    std::vector<Tensor> tensors_;
    efgs_workspace ws_{};
};

inline void check_status(int rc) {
    if (rc == EFGS_OK) return;
    const char* message = efgs_last_error();
    TORCH_CHECK(false, "efgs: ", message && *message ? message : "error", " (status ", rc, ")");
}

inline void* current_stream(at::Device device) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream(); }

inline int32_t element_type(const char* name, at::ScalarType type) {
    switch (type) {
        case at::kFloat: return EFGS_FLOAT;
        case at::kBFloat16: return EFGS_BFLOAT16;
        case at::kHalf: return EFGS_HALF;
        default: TORCH_CHECK_VALUE(false, "efgs: ", name, " must be float32, bfloat16 or float16, got ", type);
    }
}

// Scratch of a call, as much as it asks for (in one request: a region that follows the largest call so far, as the rasterizer's does
// to spare allocations, would save none and hold as much for a few rows as for the longest list).
class Scratch {
  public:
    explicit Scratch(at::Device device) : options_(at::TensorOptions().dtype(at::kByte).device(device)) {}
    static void* alloc(void* self, size_t bytes) noexcept {
        try {
            Scratch* s = static_cast<Scratch*>(self);
            s->tensors_.push_back(at::empty({static_cast<int64_t>(bytes > 0 ? bytes : 1)}, s->options_));
            return s->tensors_.back().data_ptr();
        } catch (...) {  // (out of memory: the library reports the failed allocation)
            return nullptr;
        }
    }

  private:
    at::TensorOptions options_;
    std::vector<Tensor> tensors_;
};

template <typename T>
T* pointer(const Tensor& t) {
    return t.numel() > 0 ? static_cast<T*>(t.data_ptr()) : nullptr;
}

// The gradients of a backward that is itself being differentiated (create_graph with an upstream that requires a
// gradient) hang on the upstream by an identity whose own backward raises: the kernels have no second derivatives, and a
// graph without this edge would give zeros for them. The message is the one that Python autograd functions marked
// once_differentiable give, which programs may look for.
struct FirstOrderOnly : torch::autograd::Function<FirstOrderOnly> {
    static Tensor forward(AutogradContext*, const Tensor& /*upstream*/, const Tensor& grad) { return grad.variable_data(); }  // (no view: it may be changed in place)
    static variable_list backward(AutogradContext*, variable_list) {
        TORCH_CHECK(false, "trying to differentiate twice a function that was marked with @once_differentiable");
    }
};

inline variable_list first_order_only(variable_list grads, const Tensor& upstream) {
    if (at::GradMode::is_enabled() && upstream.requires_grad())
        for (Tensor& g : grads)
            if (g.defined()) g = FirstOrderOnly::apply(upstream, g);
    return grads;
}

// The same for gradients that depend on the node's inputs too, as a loss's that is not linear in them: whenever the backward is being
// recorded, they hang on everything that the node's inputs came from, so that no path back to them passes by the refusal.
struct InputsOnce : torch::autograd::Node {
    variable_list apply(variable_list&&) override { TORCH_CHECK(false, "trying to differentiate twice a function that was marked with @once_differentiable"); }
};

// called within the node's backward
inline variable_list first_order_only_in_inputs(variable_list grads, const Tensor& upstream) {
    if (!at::GradMode::is_enabled()) return grads;
    const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node(), refusal(new InputsOnce(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges = node ? node->next_edges() : torch::autograd::edge_list{};
    if (upstream.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(upstream));
    refusal->set_next_edges(std::move(edges));
    for (Tensor& g : grads)
        if (g.defined()) torch::autograd::set_history(g, refusal);
    return grads;
}

}  // namespace efgs_torch
