// Shared parts of the encoder operators' bindings: checks of tensors, workspaces, streams, and the nodes of the autograd graph.
#pragma once
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/library.h>

#include <vector>

#include "../../include/mam_hip.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::vector<Tensor> Tensors;
typedef c10::optional<Tensor> MaybeTensor;

inline void *current_stream(const Tensor &t) { return static_cast<void *>(c10::hip::getCurrentHIPStream(t.get_device()).stream()); }

inline void check_rc(int rc, const char *what)
{
    TORCH_CHECK(rc == MAM_OK, what, " failed: ", mam_error_string(rc), " (", mam_last_error(), ")");
}

inline int type_of(const Tensor &t, const char *name)
{
    TORCH_CHECK(t.is_cuda(), name, " must be on the GPU");
    switch (t.scalar_type()) {
        case at::kFloat: return MAM_F32;
        case at::kBFloat16: return MAM_BF16;
        case at::kHalf: return MAM_F16;
        default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
    return -1;
}

inline void check_like(const Tensor &t, const Tensor &x, const char *name)
{
    TORCH_CHECK(t.device() == x.device(), name, " is on a different device");
    TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " must have the operand's type ", x.scalar_type(), ", got ", t.scalar_type());
    TORCH_CHECK(t.sizes() == x.sizes(), name, " must have the operand's shape ", x.sizes(), ", got ", t.sizes());
}

inline bool has(const MaybeTensor &t) { return t.has_value() && t->defined(); }
inline const void *ptr(const MaybeTensor &t) { return has(t) ? t->data_ptr() : nullptr; }
inline void *out_ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

inline Tensor workspace_for(size_t bytes, const Tensor &like)
{
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}

// A tensor with elements next to each other in its last dimension: itself, or a copy.
inline Tensor unit_last(const Tensor &t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

inline Tensor or_empty(const Tensor &t, const Tensor &like) { return t.defined() ? t : at::empty({0}, like.options()); }

// ---- autograd ----
// Nodes of the graph that hold what they need as members and compute what is asked of them.  A small call's host time is mostly
// autograd's: with custom functions, which keep their arguments in a dictionary and wrap every output, forward and gradient of
// layer_norm at 64 x 256 take 75 to 77 us of host time against 71 to 73 here, of dropout 48 to 50 against 46 to 47.  Every call goes
// through the dispatcher, so that fake tensors and tracing see the operators.
template <class Signature>
c10::TypedOperatorHandle<Signature> find(const char *name)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

inline bool wants(const Tensor &t) { return t.defined() && t.requires_grad(); }
inline bool wants(const MaybeTensor &t) { return t.has_value() && wants(*t); }
template <class... T>
inline bool recording(const T &...t)
{
    return at::GradMode::is_enabled() && (wants(t) || ...);
}
// A tangent would be dropped without a word.
inline bool has_tangent(const Tensor &t) { return t.defined() && t._fw_grad(0).defined(); }
inline bool has_tangent(const MaybeTensor &t) { return t.has_value() && has_tangent(*t); }
template <class... T>
inline void check_no_tangent(const char *what, const T &...t)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(t) || ...), what, " has no forward-mode derivative");
}
inline Tensor or_none(const MaybeTensor &t) { return has(t) ? *t : Tensor(); }
inline MaybeTensor maybe(const Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

struct GradNode : public torch::autograd::Node {
    std::vector<SavedVariable> saved;
    void save(const Tensor &t) { saved.emplace_back(t, false); }
    void save_output(const Tensor &t) { saved.emplace_back(t, true); }
    Tensor take(size_t i) { return saved[i].unpack(shared_from_this()); }
    void release_variables() override { saved.clear(); }
    // Gradients that are asked for with a graph of their own: the kernels' gradients have no formula for a second derivative, so going
    // through one of them is an error, not a gradient that lacks a part.
    void check_differentiated_once(const variable_list &grads, variable_list &out)
    {
        if (!at::GradMode::is_enabled()) return;
        torch::autograd::edge_list edges = torch::autograd::collect_next_edges(grads);
        for (SavedVariable &v : saved) {
            const Tensor t = v.unpack(shared_from_this());
            if (wants(t)) edges.push_back(torch::autograd::impl::gradient_edge(t));
        }
        bool any = false;
        for (const torch::autograd::Edge &e : edges) any = any || e.is_valid();
        if (!any) return;
        const auto node = std::shared_ptr<torch::autograd::Error>(
            new torch::autograd::Error("the gradient of " + name() + " is not implemented", std::move(edges)), torch::autograd::deleteNode);
        for (Tensor &t : out)
            if (t.defined()) torch::autograd::set_history(t, node);
    }
    // Saved tensors are gone once a graph that is not retained has been walked.
    void check_saved() const { TORCH_CHECK(!saved.empty(), torch::autograd::ERR_BACKWARD_TWICE); }
};

template <class N, class... T>
std::shared_ptr<N> node_of(const T &...inputs)
{
    auto node = std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
    torch::autograd::edge_list edges;
    const auto add = [&](const Tensor &t) {
        edges.push_back(t.defined() && t.requires_grad() ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge());
    };
    (add(inputs), ...);
    node->set_next_edges(std::move(edges));
    return node;
}

}  // namespace
