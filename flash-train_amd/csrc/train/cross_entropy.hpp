// What the cross entropy's host code (cross_entropy.hip) and its tile kernels (one translation unit per
// element type, cross_entropy_tiles.hpp) share.
#pragma once

#include <cstdint>

#include <hip/hip_runtime.h>

#include <flash_train/common.h>

namespace ftrain::train {

// What the device knows of the batch.
struct Head {
    int32_t valid;  // packed rows
    float scale;    // dl is kept times this power of two
    float inv_scale;
};

// One packed row: where its lse, its gradient of the loss and its target are.
struct RowInfo {
    float lse;
    float grad;      // times Head::scale
    int32_t target;  // -1: outside the classes
};

// Each row's target: of the packed rows or, without these, of every token.
struct Targets {
    const RowInfo* rows;
    const void* target;
    int64_t ignore_index, classes;
    bool wide;  // int64, else int32

    __device__ __forceinline__ int64_t given(int64_t token) const {
        return wide ? static_cast<const int64_t*>(target)[token] : static_cast<int64_t>(static_cast<const int32_t*>(target)[token]);
    }
    // -1: outside the classes.
    __device__ __forceinline__ int of(int64_t token) const {
        const int64_t y = given(token);
        return y >= 0 && y < classes ? static_cast<int>(y) : -1;
    }
    __device__ __forceinline__ int operator()(int64_t row) const { return rows != nullptr ? rows[row].target : of(row); }
};

// The products of the two passes.
enum class HeadTile {
    kLogSum,      // tokens x classes: each row's maximum and sum of exponentials over a tile's classes
    kGradLogits,  // tokens x classes: dl
    kGradHidden,  // tokens x hidden = dl w, fp32 sums of a slice of the classes
    kGradWeight,  // classes x hidden = dl^T x
    kLogits,      // tokens x classes: fp32 sums of a slice of the hidden values
};

// Up to this many tokens (16-bit types) the products are the weight's reading, and the arithmetic is free:
// the smallest tile's rows, k of the logits cut where the tiles are few, and dl kept in two adjacent rows,
// its value rounded and what that left (twice the mantissa), against two equal rows of x.  With one
// rounding the gradients of 16 tokens, where single values of dl count, were 1.6 times as far from 64 bits
// as the rounding of the result alone; of many tokens 1.4 times.
constexpr int64_t kFewTokens = 64;

// Up to this many tokens (fp32) dl's logits are summed apart (headTileFp32).
constexpr int64_t kApartTokens = 128;

struct HeadTileArgs {
    const void *a, *b;
    void* d;
    int64_t lda, ldb, ldd;
    int32_t m, n, k;
    int32_t read_m, read_n;  // what the storage of transposed operands holds; 0: m, n
    const Head* head;  // null: all of the tokens
    Targets targets;
    int32_t pair;  // kGradHidden, kGradWeight: rows of dl (and x) of each packed token (kFewTokens)
    int32_t first_class;
    // kLogSum: a pair of maximum and sum of each part of the classes and, within it, of each of `tokens`
    // rows; the logit of each row's target.
    float2* part;
    float* hit;
    int64_t tokens;
    // kGradHidden, kLogits: the k of one of gridDim.z slices, elements from one slice's sums to the next's,
    // and (kGradHidden) whether the sums of earlier classes are added to.
    int32_t k_chunk;
    int64_t slice;
    bool add;
};

// Launches the product on tiles of `rows` rows (16-bit: 256x256, 128x128, 64x128; fp32: 128x128, 64x64;
// the weight's gradient: not the last of either; kLogits: not 256x256); m counts every token, the kernels take the
// packed ones only.
void launchHeadTileFp32(HeadTile what, int rows, const HeadTileArgs& args, int slices, hipStream_t stream);
void launchHeadTileBf16(HeadTile what, int rows, const HeadTileArgs& args, int slices, hipStream_t stream);
void launchHeadTileFp16(HeadTile what, int rows, const HeadTileArgs& args, int slices, hipStream_t stream);
// kGradHidden and kGradWeight, both on tiles of 128 rows, in one launch.
void launchHeadGradientsBf16(const HeadTileArgs& hidden, int slices, const HeadTileArgs& weight, hipStream_t stream);
void launchHeadGradientsFp16(const HeadTileArgs& hidden, int slices, const HeadTileArgs& weight, hipStream_t stream);

}  // namespace ftrain::train
