// flash_train.torch's operators around a training step's products, over the C entry points of
// flash_train.h: outputs and workspaces come from torch's allocator, the work goes to the current stream.
#include "training.hpp"

#include <vector>

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <flash_train/flash_train.h>

namespace {

using at::Tensor;

FTrainNumericType numericType(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return FTRAIN_NUMERIC_TYPE_FP32;
        case at::kBFloat16: return FTRAIN_NUMERIC_TYPE_BF16;
        case at::kHalf: return FTRAIN_NUMERIC_TYPE_FP16;
        case at::kLong: return FTRAIN_NUMERIC_TYPE_INT64;
        case at::kInt: return FTRAIN_NUMERIC_TYPE_INT32;
        case at::kBool:
        case at::kByte: return FTRAIN_NUMERIC_TYPE_UINT8;
        default: TORCH_CHECK(false, "unsupported tensor type ", t.scalar_type());
    }
}

// A view of a device tensor as it lies.
FTrainStorageView view(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a device tensor");
    const bool dense = t.is_contiguous();
    return FTrainStorageView{t.data_ptr(),
                             t.sizes().data(),
                             dense ? nullptr : t.strides().data(),
                             static_cast<uint8_t>(t.dim()),
                             numericType(t),
                             static_cast<FTrainIndexType>(dense ? FTRAIN_INDEX_TYPE_CONTINUOUS : FTRAIN_INDEX_TYPE_INVALID),
                             false};
}

// A tensor of one value as an array of one.
FTrainStorageView viewOne(const Tensor& t, const char* name) {
    static const int64_t one = 1;
    FTrainStorageView v      = view(t, name);
    v.dims = &one, v.strides = nullptr, v.num_dims = 1;
    return v;
}

FTrainStorageView none() {
    static const int64_t zero = 0;
    return FTrainStorageView{nullptr, &zero, nullptr, 1, FTRAIN_NUMERIC_TYPE_UINT8, FTRAIN_INDEX_TYPE_CONTINUOUS, false};
}

void check(FTrainStatus status, const char* what) {
    TORCH_CHECK(status == FTRAIN_STATUS_SUCCESS, what, " failed with status ", static_cast<unsigned>(status), ": ",
                ftrainGetLastMessage());
}

// The device of a call: its guard, its current stream, and tensors made on it.
class Call {
  public:
    explicit Call(const Tensor& t, const char* name) : device_(deviceOf(t, name)), guard_(device_) {
        stream_ = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device_.index()).stream();
    }
    void same(const Tensor& t, const char* name) const {
        TORCH_CHECK(t.is_cuda() && t.device() == device_, name, " must be on the device of the other tensors");
    }
    // An output.  Made below the dispatcher, and the workspace below tensors: a call of the router on few
    // tokens is bound by the host, on which torch::empty takes 1 us.
    Tensor make(at::IntArrayRef sizes, at::ScalarType type) const {
        return Tensor(at::detail::empty_cuda(sizes, type, device_, c10::nullopt));
    }
    // Memory of the current stream, as a tensor's is.
    c10::DataPtr workspace(uint64_t bytes) const { return c10::GetAllocator(c10::kCUDA)->allocate(bytes); }
    hipStream_t stream() const { return stream_; }

  private:
    static c10::Device deviceOf(const Tensor& t, const char* name) {
        TORCH_CHECK(t.is_cuda(), name, " must be a device tensor");
        return t.device();
    }
    c10::Device device_;
    c10::hip::HIPGuardMasqueradingAsCUDA guard_;
    hipStream_t stream_;
};

void checkRank(const Tensor& t, const char* name, int64_t rank) {
    TORCH_CHECK(t.dim() == rank, name, " must have rank ", rank);
}

// A tensor whose rows are contiguous, copied if its own are not.
Tensor withRows(const Tensor& t) {
    return t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t
                                                                                                                : t.contiguous();
}

std::tuple<Tensor, Tensor> crossEntropyForward(const Tensor& hidden_, const Tensor& weight_, const Tensor& target_,
                                               int64_t ignore_index) {
    Call call(hidden_, "hidden");
    call.same(weight_, "weight");
    call.same(target_, "target");
    checkRank(hidden_, "hidden", 2);
    checkRank(weight_, "weight", 2);
    checkRank(target_, "target", 1);
    const Tensor hidden = withRows(hidden_), weight = withRows(weight_), target = target_.contiguous();
    Tensor loss = call.make({hidden.size(0)}, at::kFloat), lse = call.make({hidden.size(0)}, at::kFloat);
    uint64_t bytes = 0;
    check(ftrainLinearCrossEntropyWorkspaceBytes(view(hidden, "hidden"), view(weight, "weight"), false, &bytes),
          "ftrainLinearCrossEntropyWorkspaceBytes");
    const c10::DataPtr workspace = call.workspace(bytes);
    check(ftrainLinearCrossEntropy(view(hidden, "hidden"), view(weight, "weight"), view(target, "target"),
                                   view(loss, "loss"), view(lse, "lse"), ignore_index, workspace.get(), bytes,
                                   call.stream()),
          "ftrainLinearCrossEntropy");
    return {loss, lse};
}

std::tuple<Tensor, Tensor> crossEntropyBackward(const Tensor& grad_loss_, const Tensor& hidden_, const Tensor& weight_,
                                                const Tensor& target_, const Tensor& lse_, int64_t ignore_index) {
    Call call(hidden_, "hidden");
    call.same(weight_, "weight");
    call.same(target_, "target");
    call.same(grad_loss_, "grad_loss");
    call.same(lse_, "lse");
    checkRank(hidden_, "hidden", 2);
    checkRank(weight_, "weight", 2);
    checkRank(target_, "target", 1);
    const Tensor hidden = withRows(hidden_), weight = withRows(weight_), target = target_.contiguous();
    const Tensor grad_loss = grad_loss_.contiguous(), lse = lse_.contiguous();
    Tensor grad_hidden = call.make(hidden.sizes(), hidden.scalar_type());
    Tensor grad_weight = call.make(weight.sizes(), weight.scalar_type());
    uint64_t bytes     = 0;
    check(ftrainLinearCrossEntropyWorkspaceBytes(view(hidden, "hidden"), view(weight, "weight"), true, &bytes),
          "ftrainLinearCrossEntropyWorkspaceBytes");
    const c10::DataPtr workspace = call.workspace(bytes);
    check(ftrainLinearCrossEntropyBackward(view(grad_loss, "grad_loss"), view(hidden, "hidden"), view(weight, "weight"),
                                           view(target, "target"), view(lse, "lse"), view(grad_hidden, "grad_hidden"),
                                           view(grad_weight, "grad_weight"), ignore_index, workspace.get(), bytes,
                                           call.stream()),
          "ftrainLinearCrossEntropyBackward");
    return {grad_hidden, grad_weight};
}

// The mask as the entry points take it: one byte a row, or none.
FTrainStorageView maskView(const Call& call, const c10::optional<Tensor>& mask, Tensor& keep) {
    if (!mask.has_value()) return none();
    call.same(*mask, "mask");
    TORCH_CHECK(mask->scalar_type() == at::kBool, "mask must be bool");
    keep = mask->contiguous();
    return keep.numel() == 0 ? none() : view(keep, "mask");
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> routeForward(const Tensor& logits_, int64_t top_k, bool normalize,
                                                                        const c10::optional<Tensor>& mask) {
    Call call(logits_, "logits");
    checkRank(logits_, "logits", 2);
    const Tensor logits = withRows(logits_);
    const int64_t rows = logits.size(0), n = logits.size(1);
    TORCH_CHECK(top_k >= 1, "top_k must be positive");
    Tensor mask_dense;
    const FTrainStorageView mask_view = maskView(call, mask, mask_dense);
    TORCH_CHECK(!mask.has_value() || (mask->dim() == 1 && mask->size(0) == rows), "mask must hold one value a row");
    Tensor experts = call.make({rows, top_k}, at::kInt), gates = call.make({rows, top_k}, at::kFloat);
    Tensor slots = call.make({rows, top_k}, at::kInt), counts = call.make({n}, at::kInt);
    Tensor routed = call.make({1}, at::kInt), loss = call.make({}, at::kFloat);
    uint64_t bytes = 0;
    check(ftrainMoeRouteWorkspaceBytes(view(logits, "logits"), &bytes), "ftrainMoeRouteWorkspaceBytes");
    const c10::DataPtr workspace = call.workspace(bytes);
    check(ftrainMoeRoute(view(logits, "logits"), mask_view, view(experts, "experts"), view(gates, "gates"),
                         view(slots, "slots"), view(counts, "counts"), view(routed, "routed"), viewOne(loss, "loss"), normalize,
                         workspace.get(), bytes, call.stream()),
          "ftrainMoeRoute");
    return {experts, gates, slots, counts, routed, loss};
}

Tensor routeBackward(const Tensor& grad_gates_, const Tensor& grad_loss_, const Tensor& logits_, const Tensor& experts_,
                     const Tensor& counts_, const Tensor& routed_, bool normalize, const c10::optional<Tensor>& mask) {
    Call call(logits_, "logits");
    checkRank(logits_, "logits", 2);
    for (const auto& [t, name] : {std::pair<const Tensor&, const char*>{grad_gates_, "grad_gates"}, {grad_loss_, "grad_loss"},
                                  {experts_, "experts"}, {counts_, "counts"}, {routed_, "routed"}})
        call.same(t, name);
    const Tensor logits = withRows(logits_), experts = experts_.contiguous(), counts = counts_.contiguous();
    const Tensor grad_gates = grad_gates_.contiguous(), routed = routed_.contiguous();
    TORCH_CHECK(grad_loss_.numel() == 1, "grad_loss must hold one value");
    Tensor mask_dense;
    const FTrainStorageView mask_view = maskView(call, mask, mask_dense);
    TORCH_CHECK(!mask.has_value() || (mask->dim() == 1 && mask->size(0) == logits.size(0)), "mask must hold one value a row");
    Tensor grad_logits = call.make(logits.sizes(), logits.scalar_type());
    check(ftrainMoeRouteBackward(view(grad_gates, "grad_gates"), viewOne(grad_loss_, "grad_loss"), view(logits, "logits"), mask_view,
                                 view(experts, "experts"), view(counts, "counts"), view(routed, "routed"),
                                 view(grad_logits, "grad_logits"), normalize, call.stream()),
          "ftrainMoeRouteBackward");
    return grad_logits;
}

Tensor clipGradNorm(const std::vector<Tensor>& grads, double max_norm, double eps,
                    const c10::optional<std::vector<Tensor>>& out) {
    TORCH_CHECK(!grads.empty(), "there must be a gradient at least");
    Call call(grads[0], "grads[0]");
    TORCH_CHECK(!out.has_value() || out->size() == grads.size(), "out must hold one tensor for each gradient");
    // Scaling is elementwise, so a dense tensor is taken in the order in which it lies in memory.
    std::vector<int64_t> counts(grads.size());
    std::vector<FTrainStorageView> in_views(grads.size()), out_views(grads.size());
    for (std::size_t i = 0; i < grads.size(); ++i) {
        const Tensor& g = grads[i];
        const Tensor& o = out.has_value() ? (*out)[i] : g;
        call.same(g, "every gradient");
        call.same(o, "every output");
        TORCH_CHECK(g.is_non_overlapping_and_dense(), "grads[", i, "] must be dense");
        TORCH_CHECK(o.sizes() == g.sizes() && o.strides() == g.strides() && o.scalar_type() == g.scalar_type(), "out[", i,
                    "] must be like grads[", i, "]");
        counts[i]    = g.numel();
        in_views[i]  = FTrainStorageView{g.data_ptr(), &counts[i], nullptr, 1, numericType(g), FTRAIN_INDEX_TYPE_CONTINUOUS, false};
        out_views[i] = in_views[i];
        out_views[i].memory = o.data_ptr();
    }
    Tensor norm    = call.make({}, at::kFloat);
    uint64_t bytes = 0;
    check(ftrainClipGradNormWorkspaceBytes(&bytes), "ftrainClipGradNormWorkspaceBytes");
    const c10::DataPtr workspace = call.workspace(bytes);
    check(ftrainClipGradNorm(in_views.data(), out_views.data(), static_cast<uint32_t>(grads.size()), viewOne(norm, "norm"),
                             static_cast<float>(max_norm), static_cast<float>(eps), workspace.get(), bytes,
                             call.stream()),
          "ftrainClipGradNorm");
    return norm;
}

}  // namespace

void bindTraining(py::module_& m) {
    m.def("linear_cross_entropy_forward", &crossEntropyForward,
          "(loss, lse) of every token of softmax cross entropy over hidden @ weight.T", py::arg("hidden"), py::arg("weight"),
          py::arg("target"), py::arg("ignore_index") = -100);
    m.def("linear_cross_entropy_backward", &crossEntropyBackward, "(grad_hidden, grad_weight)", py::arg("grad_loss"),
          py::arg("hidden"), py::arg("weight"), py::arg("target"), py::arg("lse"), py::arg("ignore_index") = -100);
    m.def("moe_route_forward", &routeForward, "(experts, gates, slots, counts, routed, balance_loss)", py::arg("logits"),
          py::arg("top_k"), py::arg("normalize") = false, py::arg("mask") = py::none());
    m.def("moe_route_backward", &routeBackward, "grad_logits", py::arg("grad_gates"), py::arg("grad_loss"), py::arg("logits"),
          py::arg("experts"), py::arg("counts"), py::arg("routed"), py::arg("normalize") = false, py::arg("mask") = py::none());
    m.def("clip_grad_norm", &clipGradNorm,
          "The global norm; the gradients times min(1, max_norm / (norm + eps)) in place or to out", py::arg("grads"),
          py::arg("max_norm"), py::arg("eps") = 1e-6, py::arg("out") = py::none());
}
