// The C entry points of the operators around a training step's products
// (include/flash_train/flash_train.h): each checks its views, then launches
// (ft/train.hpp).  They have no counterpart in the reference.
#include <cmath>
#include <string>

#include <flash_train/flash_train.h>

#include "ft/handles.hpp"
#include "ft/trace.hpp"
#include "ft/train.hpp"

namespace ftrain {
namespace {

using train::Rows;

// Checks arguments on behalf of one entry point; every failure names it and the argument.
class Checker {
  public:
    explicit Checker(const char* fn) : fn_(fn) {}

    template <class... A>
    [[noreturn]] void fail(FTrainStatus status, const char* fmt, A... args) const {
        raise(status, (std::string("%s: ") + fmt).c_str(), fn_, args...);
    }

    StorageView device(const FTrainStorageView& v, const char* name, std::size_t rank) const {
        StorageView view(v);
        if (view.isHost()) fail(FTRAIN_STATUS_INVALID_ARGUMENT, "%s must be in device memory", name);
        if (view.rank() != rank)
            fail(FTRAIN_STATUS_INVALID_ARGUMENT, "%s must have rank %zu, got %zu", name, rank, view.rank());
        if (view.indexType() != FTRAIN_INDEX_TYPE_CONTINUOUS && view.indexType() != FTRAIN_INDEX_TYPE_INVALID)
            fail(FTRAIN_STATUS_UNSUPPORTED, "%s must be continuous or strided", name);
        return view;
    }

    void type(const StorageView& v, const char* name, FTrainNumericType type) const {
        if (v.numericType() != type)
            fail(FTRAIN_STATUS_UNSUPPORTED, "%s has numeric type %u, needs %u", name, unsigned(v.numericType()), unsigned(type));
    }

    void address(const StorageView& v, const char* name, std::size_t bytes, bool empty) const {
        if (v.memory() == nullptr && !empty) fail(FTRAIN_STATUS_INVALID_ARGUMENT, "%s must not be null", name);
        if (reinterpret_cast<uintptr_t>(v.memory()) % bytes != 0)
            fail(FTRAIN_STATUS_UNSUPPORTED, "%s is not aligned to its element size", name);
    }

    // A matrix of fp32, bf16 or fp16 with contiguous rows.
    Rows rows(const FTrainStorageView& v, const char* name, FTrainNumericType& type) const {
        const StorageView view = device(v, name, 2);
        type                   = view.numericType();
        if (type != FTRAIN_NUMERIC_TYPE_FP32 && type != FTRAIN_NUMERIC_TYPE_BF16 && type != FTRAIN_NUMERIC_TYPE_FP16)
            fail(FTRAIN_STATUS_UNSUPPORTED, "%s must be fp32, bf16 or fp16", name);
        Rows r{view.memory(), view.dims()[0], view.dims()[1], view.dims()[1]};
        if (!view.strides().empty()) {
            r.ld = view.strides()[0];
            if (r.cols > 1 && view.strides()[1] != 1) fail(FTRAIN_STATUS_UNSUPPORTED, "%s must have contiguous rows", name);
            if (r.rows <= 1) r.ld = std::max(r.ld, r.cols);
            if (r.ld < r.cols) fail(FTRAIN_STATUS_UNSUPPORTED, "%s has rows that overlap", name);
        }
        if (r.ld > (int64_t(1) << 40)) fail(FTRAIN_STATUS_UNSUPPORTED, "%s has too large a row stride", name);
        address(view, name, train::elementBytes(type), r.rows == 0 || r.cols == 0);
        return r;
    }

    Rows like(const FTrainStorageView& v, const char* name, const Rows& shape, FTrainNumericType type) const {
        FTrainNumericType t;
        const Rows r = rows(v, name, t);
        if (t != type) fail(FTRAIN_STATUS_UNSUPPORTED, "%s has numeric type %u, needs %u", name, unsigned(t), unsigned(type));
        if (r.rows != shape.rows || r.cols != shape.cols)
            fail(FTRAIN_STATUS_INVALID_ARGUMENT, "%s must be %lld x %lld", name, (long long)shape.rows, (long long)shape.cols);
        return r;
    }

    // A dense array of `dims` elements (any rank the view gives must match).
    void* dense(const FTrainStorageView& v, const char* name, std::initializer_list<int64_t> dims, FTrainNumericType t,
                std::size_t bytes) const {
        const StorageView view = device(v, name, dims.size());
        type(view, name, t);
        std::size_t i = dims.size();
        int64_t run   = 1;
        for (auto it = std::rbegin(dims); it != std::rend(dims); ++it) {
            --i;
            if (view.dims()[i] != *it)
                fail(FTRAIN_STATUS_INVALID_ARGUMENT, "%s has size %lld in dimension %zu, needs %lld", name,
                     (long long)view.dims()[i], i, (long long)*it);
            if (!view.strides().empty() && *it > 1 && view.strides()[i] != run)
                fail(FTRAIN_STATUS_UNSUPPORTED, "%s must be dense", name);
            run *= *it;
        }
        address(view, name, bytes, run == 0);
        return view.memory();
    }

    void workspace(const void* memory, uint64_t bytes, uint64_t need) const {
        if (bytes < need || (need > 0 && memory == nullptr))
            fail(FTRAIN_STATUS_INVALID_ARGUMENT, "the workspace holds %llu bytes, needs %llu", (unsigned long long)bytes,
                 (unsigned long long)need);
        if (reinterpret_cast<uintptr_t>(memory) % 256 != 0)
            fail(FTRAIN_STATUS_INVALID_ARGUMENT, "the workspace must be aligned to 256 bytes");
    }

  private:
    const char* fn_;
};

// Tokens, classes, experts: whole numbers of 31 bits, with room to round up to tiles.
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 1024;
// Leading dimensions of the cross entropy's products: offsets within a tile stay below 2^32 bytes.
constexpr int64_t kMaxHidden = int64_t(1) << 20;

train::CrossEntropy crossEntropyProblem(const Checker& check, const FTrainStorageView& hidden,
                                        const FTrainStorageView& weight) {
    train::CrossEntropy p{};
    FTrainNumericType weight_type;
    p.hidden = check.rows(hidden, "hidden", p.type);
    p.weight = check.rows(weight, "weight", weight_type);
    if (weight_type != p.type) check.fail(FTRAIN_STATUS_UNSUPPORTED, "hidden and weight must have one numeric type");
    if (p.hidden.cols != p.weight.cols)
        check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "hidden has %lld columns, weight %lld", (long long)p.hidden.cols,
                   (long long)p.weight.cols);
    if (p.hidden.cols == 0 || p.weight.rows == 0)
        check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "there must be at least one class and one hidden value");
    if (p.hidden.rows > kMaxRows || p.weight.rows > kMaxRows)
        check.fail(FTRAIN_STATUS_UNSUPPORTED, "at most %lld tokens and classes are supported", (long long)kMaxRows);
    if (p.hidden.cols > kMaxHidden || p.weight.ld > kMaxHidden)
        check.fail(FTRAIN_STATUS_UNSUPPORTED, "hidden values and the weight's row stride go to %lld", (long long)kMaxHidden);
    return p;
}

void crossEntropyTarget(const Checker& check, train::CrossEntropy& p, const FTrainStorageView& target, int64_t ignore_index) {
    p.target_wide  = target.numeric_type == FTRAIN_NUMERIC_TYPE_INT64;
    p.target       = check.dense(target, "target", {p.hidden.rows},
                                 p.target_wide ? FTRAIN_NUMERIC_TYPE_INT64 : FTRAIN_NUMERIC_TYPE_INT32, p.target_wide ? 8 : 4);
    p.ignore_index = ignore_index;
}

train::MoeRoute routeProblem(const Checker& check, const FTrainStorageView& logits, const FTrainStorageView& experts) {
    train::MoeRoute p{};
    p.logits              = check.rows(logits, "logits", p.type);
    const StorageView out = check.device(experts, "experts", 2);
    const int64_t top_k   = out.dims()[1];
    if (p.logits.cols < 1 || p.logits.cols > train::kMaxExperts)
        check.fail(FTRAIN_STATUS_UNSUPPORTED, "1 to %d experts are supported, got %lld", train::kMaxExperts, (long long)p.logits.cols);
    if (top_k < 1 || top_k > train::kMaxTopK || top_k > p.logits.cols)
        check.fail(FTRAIN_STATUS_UNSUPPORTED, "a token takes 1 to %d of its experts, got %lld of %lld", train::kMaxTopK,
                   (long long)top_k, (long long)p.logits.cols);
    if (p.logits.rows > kMaxRows / top_k)
        check.fail(FTRAIN_STATUS_UNSUPPORTED, "at most %lld choices are supported", (long long)kMaxRows);
    p.top_k   = static_cast<int>(top_k);
    p.experts = static_cast<int32_t*>(check.dense(experts, "experts", {p.logits.rows, top_k}, FTRAIN_NUMERIC_TYPE_INT32, 4));
    return p;
}

void routeCommon(const Checker& check, train::MoeRoute& p, const FTrainStorageView& mask, const FTrainStorageView& counts,
                 const FTrainStorageView& routed, bool normalize) {
    if (mask.memory != nullptr)
        p.mask = static_cast<const uint8_t*>(check.dense(mask, "mask", {p.logits.rows}, FTRAIN_NUMERIC_TYPE_UINT8, 1));
    p.counts    = static_cast<int32_t*>(check.dense(counts, "counts", {p.logits.cols}, FTRAIN_NUMERIC_TYPE_INT32, 4));
    p.routed    = static_cast<int32_t*>(check.dense(routed, "routed", {1}, FTRAIN_NUMERIC_TYPE_INT32, 4));
    p.normalize = normalize;
}

float* floats(const Checker& check, const FTrainStorageView& v, const char* name, std::initializer_list<int64_t> dims) {
    return static_cast<float*>(check.dense(v, name, dims, FTRAIN_NUMERIC_TYPE_FP32, 4));
}

}  // namespace
}  // namespace ftrain

using namespace ftrain;

extern "C" {

FTrainStatus ftrainLinearCrossEntropyWorkspaceBytes(FTrainStorageView hidden, FTrainStorageView weight, bool backward,
                                                    uint64_t* workspace_bytes) {
    return guarded([&] {
        const Checker check("ftrainLinearCrossEntropyWorkspaceBytes");
        if (workspace_bytes == nullptr) check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "workspace_bytes output must not be null");
        *workspace_bytes = train::crossEntropyWorkspace(crossEntropyProblem(check, hidden, weight), backward);
    });
}

FTrainStatus ftrainLinearCrossEntropy(FTrainStorageView hidden, FTrainStorageView weight, FTrainStorageView target,
                                      FTrainStorageView loss, FTrainStorageView lse, int64_t ignore_index, void* workspace,
                                      uint64_t workspace_bytes, FTrainStream stream) {
    TraceRange trace("ftrainLinearCrossEntropy");
    return guarded([&] {
        const Checker check("ftrainLinearCrossEntropy");
        train::CrossEntropy p = crossEntropyProblem(check, hidden, weight);
        crossEntropyTarget(check, p, target, ignore_index);
        p.loss = floats(check, loss, "loss", {p.hidden.rows});
        p.lse  = floats(check, lse, "lse", {p.hidden.rows});
        check.workspace(workspace, workspace_bytes, train::crossEntropyWorkspace(p, false));
        train::crossEntropyForward(p, workspace, stream);
    });
}

FTrainStatus ftrainLinearCrossEntropyBackward(FTrainStorageView grad_loss, FTrainStorageView hidden, FTrainStorageView weight,
                                              FTrainStorageView target, FTrainStorageView lse, FTrainStorageView grad_hidden,
                                              FTrainStorageView grad_weight, int64_t ignore_index, void* workspace,
                                              uint64_t workspace_bytes, FTrainStream stream) {
    TraceRange trace("ftrainLinearCrossEntropyBackward");
    return guarded([&] {
        const Checker check("ftrainLinearCrossEntropyBackward");
        train::CrossEntropy p = crossEntropyProblem(check, hidden, weight);
        crossEntropyTarget(check, p, target, ignore_index);
        p.grad_loss   = floats(check, grad_loss, "grad_loss", {p.hidden.rows});
        p.lse         = floats(check, lse, "lse", {p.hidden.rows});
        p.grad_hidden = check.like(grad_hidden, "grad_hidden", p.hidden, p.type);
        p.grad_weight = check.like(grad_weight, "grad_weight", p.weight, p.type);
        if (p.grad_weight.ld > kMaxHidden)
            check.fail(FTRAIN_STATUS_UNSUPPORTED, "grad_weight's row stride goes to %lld", (long long)kMaxHidden);
        check.workspace(workspace, workspace_bytes, train::crossEntropyWorkspace(p, true));
        train::crossEntropyBackward(p, workspace, stream);
    });
}

FTrainStatus ftrainMoeRouteWorkspaceBytes(FTrainStorageView logits, uint64_t* workspace_bytes) {
    return guarded([&] {
        const Checker check("ftrainMoeRouteWorkspaceBytes");
        if (workspace_bytes == nullptr) check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "workspace_bytes output must not be null");
        FTrainNumericType type;
        const Rows r     = check.rows(logits, "logits", type);
        *workspace_bytes = train::moeRouteWorkspace(r.rows, r.cols);
    });
}

FTrainStatus ftrainMoeRoute(FTrainStorageView logits, FTrainStorageView mask, FTrainStorageView experts, FTrainStorageView gates,
                            FTrainStorageView slots, FTrainStorageView counts, FTrainStorageView routed,
                            FTrainStorageView balance_loss, bool normalize, void* workspace, uint64_t workspace_bytes,
                            FTrainStream stream) {
    TraceRange trace("ftrainMoeRoute");
    return guarded([&] {
        const Checker check("ftrainMoeRoute");
        train::MoeRoute p = routeProblem(check, logits, experts);
        routeCommon(check, p, mask, counts, routed, normalize);
        p.gates        = floats(check, gates, "gates", {p.logits.rows, p.top_k});
        p.slots        = static_cast<int32_t*>(
            check.dense(slots, "slots", {p.logits.rows, p.top_k}, FTRAIN_NUMERIC_TYPE_INT32, 4));
        p.balance_loss = floats(check, balance_loss, "balance_loss", {1});
        check.workspace(workspace, workspace_bytes, train::moeRouteWorkspace(p.logits.rows, p.logits.cols));
        train::moeRouteForward(p, workspace, stream);
    });
}

FTrainStatus ftrainMoeRouteBackward(FTrainStorageView grad_gates, FTrainStorageView grad_loss, FTrainStorageView logits,
                                    FTrainStorageView mask, FTrainStorageView experts, FTrainStorageView counts,
                                    FTrainStorageView routed, FTrainStorageView grad_logits, bool normalize,
                                    FTrainStream stream) {
    TraceRange trace("ftrainMoeRouteBackward");
    return guarded([&] {
        const Checker check("ftrainMoeRouteBackward");
        train::MoeRoute p = routeProblem(check, logits, experts);
        routeCommon(check, p, mask, counts, routed, normalize);
        p.grad_gates  = floats(check, grad_gates, "grad_gates", {p.logits.rows, p.top_k});
        p.grad_loss   = floats(check, grad_loss, "grad_loss", {1});
        p.grad_logits = check.like(grad_logits, "grad_logits", p.logits, p.type);
        train::moeRouteBackward(p, stream);
    });
}

FTrainStatus ftrainClipGradNormWorkspaceBytes(uint64_t* workspace_bytes) {
    return guarded([&] {
        const Checker check("ftrainClipGradNormWorkspaceBytes");
        if (workspace_bytes == nullptr) check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "workspace_bytes output must not be null");
        *workspace_bytes = train::clipWorkspace();
    });
}

FTrainStatus ftrainClipGradNorm(const FTrainStorageView grads[], const FTrainStorageView outputs[], uint32_t num_grads,
                                FTrainStorageView norm, float max_norm, float eps, void* workspace, uint64_t workspace_bytes,
                                FTrainStream stream) {
    TraceRange trace("ftrainClipGradNorm");
    return guarded([&] {
        const Checker check("ftrainClipGradNorm");
        if (num_grads > 0 && grads == nullptr) check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "grads must not be null");
        if (!(max_norm >= 0.f) || !(eps >= 0.f))
            check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "max_norm and eps must not be negative");
        std::vector<train::ClipTensor> tensors(num_grads);
        for (uint32_t i = 0; i < num_grads; ++i) {
            const FTrainStorageView* views[2] = {&grads[i], outputs != nullptr ? &outputs[i] : &grads[i]};
            for (int side = 0; side < 2; ++side) {
                const StorageView v(*views[side]);
                const char* const name = side == 0 ? "grads" : "outputs";
                if (v.isHost()) check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "%s[%u] must be in device memory", name, i);
                const FTrainNumericType t = v.numericType();
                if (t != FTRAIN_NUMERIC_TYPE_FP32 && t != FTRAIN_NUMERIC_TYPE_BF16 && t != FTRAIN_NUMERIC_TYPE_FP16)
                    check.fail(FTRAIN_STATUS_UNSUPPORTED, "%s[%u] must be fp32, bf16 or fp16", name, i);
                if (v.indexType() != FTRAIN_INDEX_TYPE_CONTINUOUS)
                    check.fail(FTRAIN_STATUS_UNSUPPORTED, "%s[%u] must be continuous", name, i);
                uint64_t count = 1;
                for (const int64_t d : v.dims())
                    if (__builtin_mul_overflow(count, static_cast<uint64_t>(d), &count) || count > (uint64_t(1) << 45))
                        check.fail(FTRAIN_STATUS_OVERFLOW, "%s[%u] has too many elements", name, i);
                if (v.memory() == nullptr && count != 0)
                    check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "%s[%u] must not be null", name, i);
                if (reinterpret_cast<uintptr_t>(v.memory()) % train::elementBytes(t) != 0)
                    check.fail(FTRAIN_STATUS_UNSUPPORTED, "%s[%u] is not aligned to its element size", name, i);
                if (side == 0) {
                    tensors[i] = train::ClipTensor{v.memory(), nullptr, count, t};
                } else {
                    if (count != tensors[i].count || t != tensors[i].type)
                        check.fail(FTRAIN_STATUS_INVALID_ARGUMENT, "outputs[%u] must be like grads[%u]", i, i);
                    tensors[i].out = v.memory();
                }
            }
        }
        float* const out = floats(check, norm, "norm", {1});
        check.workspace(workspace, workspace_bytes, train::clipWorkspace());
        train::clipGradNorm(tensors.data(), tensors.size(), out, max_norm, eps, workspace, stream);
    });
}

}  // extern "C"
