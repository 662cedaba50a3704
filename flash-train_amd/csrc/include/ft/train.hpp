// The operators around a training step's products: the output head's cross
// entropy, the router of a mixture of experts, and gradient clipping.  Each
// function launches its kernels on `stream` and returns; arguments have been
// checked by the C entry points (api/train_api.cpp), which also say what each
// operator computes (include/flash_train/flash_train.h).
#pragma once

#include <cstddef>
#include <cstdint>

#include <hip/hip_runtime.h>

#include <flash_train/common.h>

#include "ft/error.hpp"

namespace ftrain::train {

inline std::size_t elementBytes(FTrainNumericType t) { return t == FTRAIN_NUMERIC_TYPE_FP32 ? 4 : 2; }

// Launches `kernel` with the arguments it declares and `lds` bytes besides its own; a failed launch raises
// INTERNAL_ERROR.
template <class... P>
void launchWithLds(void (*kernel)(P...), const char* name, dim3 grid, dim3 block, size_t lds, hipStream_t stream, P... args) {
    void* pointers[] = {static_cast<void*>(&args)...};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, pointers, lds, stream);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        raise(FTRAIN_STATUS_INTERNAL_ERROR, "%s launch failed: %s", name, hipGetErrorString(e));
    }
}
template <class... P>
void launch(void (*kernel)(P...), const char* name, dim3 grid, dim3 block, hipStream_t stream, P... args) {
    launchWithLds(kernel, name, grid, block, 0, stream, args...);
}

// A device matrix whose rows are contiguous, `ld` elements apart.
struct Rows {
    void* data;
    int64_t rows, cols, ld;
};

struct CrossEntropy {
    FTrainNumericType type;  // of hidden, weight and their gradients
    Rows hidden, weight;
    const void* target;
    bool target_wide;  // int64, else int32
    int64_t ignore_index;
    float* lse;  // forward: written; backward: read
    // forward
    float* loss;
    // backward
    const float* grad_loss;
    Rows grad_hidden, grad_weight;
};
uint64_t crossEntropyWorkspace(const CrossEntropy& p, bool backward);
void crossEntropyForward(const CrossEntropy& p, void* workspace, hipStream_t stream);
void crossEntropyBackward(const CrossEntropy& p, void* workspace, hipStream_t stream);

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK    = 32;

struct MoeRoute {
    FTrainNumericType type;  // of the logits and their gradient
    Rows logits;
    int top_k;
    bool normalize;
    const uint8_t* mask;  // null: every row counts
    int32_t* experts;     // rows x top_k, as gates and slots
    int32_t* counts;      // one of each expert
    int32_t* routed;      // one value
    // forward
    float* gates;
    int32_t* slots;
    float* balance_loss;
    // backward
    const float* grad_gates;
    const float* grad_loss;
    Rows grad_logits;
};
uint64_t moeRouteWorkspace(int64_t rows, int64_t experts);
void moeRouteForward(const MoeRoute& p, void* workspace, hipStream_t stream);
void moeRouteBackward(const MoeRoute& p, hipStream_t stream);

struct ClipTensor {
    const void* in;
    void* out;
    uint64_t count;
    FTrainNumericType type;
};
uint64_t clipWorkspace();
void clipGradNorm(const ClipTensor* tensors, std::size_t n, float* norm, float max_norm, float eps, void* workspace,
                  hipStream_t stream);

}  // namespace ftrain::train
