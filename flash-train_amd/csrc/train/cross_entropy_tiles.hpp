// The cross entropy's products on the GEMM's tiles (gemm/pingpong_tile.hpp for 16-bit types,
// gemm/dma32_tile.hpp for fp32), with the ends below in place of d = alpha acc + beta c.
#pragma once

#include "../gemm/dma32_tile.hpp"
#include "../gemm/pingpong_tile.hpp"
#include "cross_entropy.hpp"
#include "device.hpp"
#include "ft/train.hpp"

namespace ftrain::train {

// exp(x) as 2^(x log2 e): the product's rounding is off by |x| 2^-24 of the result, less than what the
// logits' own sums are.
__device__ __forceinline__ float expFast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// A row's largest logit and sum of exponentials over the N * LANES classes that its lanes hold.
template <int N, int LANES>
struct LogSumEnd {
    const RowInfo* rows;
    float2* part;
    float* hit;
    int parts, first_class;

    __device__ __forceinline__ void operator()(int row, int col, float (&v)[N], bool inside, int left) const {
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            if (e >= left) v[e] = -INFINITY;
            top = fmaxf(top, v[e]);
        }
        top       = groupMax<LANES>(top);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < N; ++e) sum += e < left ? expFast(v[e] - top) : 0.f;
        sum = groupSum<LANES>(sum);
        if (!inside) return;
        const int at = rows[row].target - first_class - col;
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e == at && e < left) hit[row] = v[e];
        // (A group may lie past the classes.)
        if (threadIdx.x % LANES == 0 && left > 0)
            part[static_cast<int64_t>(row) * parts + (first_class + col) / (N * LANES)] = make_float2(top, sum);
    }
};

// dl in the operands' type: g (exp(l - lse) - [the target]), zeros in the padding past the classes.
template <class T, int N>
struct GradLogitsEnd {
    const RowInfo* rows;
    T* d;
    int64_t ldd;
    int padded, first_class;

    __device__ __forceinline__ void operator()(int row, int col, float (&v)[N], bool inside, int left) const {
        if (!inside || col >= padded) return;
        const RowInfo r = rows[row];
        const int at    = r.target - first_class - col;
        const float g   = r.target < 0 ? NAN : r.grad;
        typedef T vec __attribute__((ext_vector_type(N)));
        vec out;
#pragma unroll
        for (int e = 0; e < N; ++e)
            out[e] = static_cast<T>(e < left ? (expFast(v[e] - r.lse) - (e == at ? 1.f : 0.f)) * g : 0.f);
        *reinterpret_cast<vec*>(d + row * ldd + col) = out;
    }
};

// fp32 dw: rows of any address.
struct GradWeightEnd {
    float* d;
    int64_t ldd;

    __device__ __forceinline__ void operator()(int row, int col, float (&v)[4], bool inside, int left) const {
        if (!inside) return;
        float* const to = d + row * ldd + col;
        if (left >= 4) {
            *reinterpret_cast<Pack<float>*>(to) = Pack<float>{v[0], v[1], v[2], v[3]};
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < left) to[e] = v[e];
        }
    }
};

// Of the launch's parameters, those of this workgroup's tile; false: no such tile (fewer rows are
// packed than tokens).
template <HeadTile WHAT, class P>
__device__ __forceinline__ bool tileProblem(const HeadTileArgs& h, P& p, int size, int tile_cols) {
    const int valid = h.head->valid;
    p.m = h.m, p.n = h.n, p.k = h.k;
    p.lda = h.lda, p.ldb = h.ldb, p.ldd = p.ldc = h.ldd;
    p.alpha = p.beta = 1.f;
    p.c              = nullptr;
    if constexpr (WHAT == HeadTile::kGradWeight)
        p.k = min(p.k, valid);
    else
        p.m = min(p.m, valid);
    p.tiles_m = (p.m + size - 1) / size;
    p.tiles_n = (p.n + tile_cols - 1) / tile_cols;
    return static_cast<int>(blockIdx.x) < p.tiles_m * p.tiles_n;
}

template <bool BF16, HeadTile WHAT>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2))) void headTileHalf(HeadTileArgs h) {
    using T = std::conditional_t<BF16, bf16, fp16>;
    gemm::HalfGemmParams p{};
    if (!tileProblem<WHAT>(h, p, 256, 256)) return;
    p.a = h.a, p.b = h.b, p.d = h.d;
    using gemm::ppdev::half_gemm_pp_tile;
    using gemm::ppdev::kBand;
    if constexpr (WHAT == HeadTile::kLogSum) {
        half_gemm_pp_tile<BF16, false, true>(p, blockIdx.x, kBand,
                                             LogSumEnd<8, 32>{h.rows, h.part, h.hit, h.parts, h.first_class});
    } else if constexpr (WHAT == HeadTile::kGradLogits) {
        half_gemm_pp_tile<BF16, false, true>(
            p, blockIdx.x, kBand,
            GradLogitsEnd<T, 8>{h.rows, static_cast<T*>(h.d), h.ldd, (h.n + 7) & ~7, h.first_class});
    } else if constexpr (WHAT == HeadTile::kGradHidden) {
        const int first = blockIdx.z * h.k_chunk;
        p.a             = static_cast<const T*>(h.a) + first;
        p.b             = static_cast<const T*>(h.b) + first * h.ldb;
        p.k             = max(0, min(h.k_chunk, h.k - first));
        p.d             = static_cast<float*>(h.d) + blockIdx.z * h.slice;
        if (h.add) p.c = p.d;
        half_gemm_pp_tile<BF16, false, false>(p, blockIdx.x, kBand);
    } else {
        p.alpha   = h.head->inv_scale;
        p.cd_half = 1;
        half_gemm_pp_tile<BF16, true, false>(p, blockIdx.x, kBand, gemm::ppdev::StoreTile{}, h.read_m, h.read_n);
    }
}

template <HeadTile WHAT>
__global__ __launch_bounds__(256, 2) void headTileFp32(HeadTileArgs h) {
    gemm::GemmParams p{};
    if (!tileProblem<WHAT>(h, p, 128, 128)) return;
    p.a = static_cast<const float*>(h.a), p.b = static_cast<const float*>(h.b), p.d = static_cast<float*>(h.d);
    using gemm::d32::fp32_gemm_dma_tile;
    using gemm::d32::StoreTile;
    constexpr int kFold = 16;
    if constexpr (WHAT == HeadTile::kLogSum) {
        const LogSumEnd<4, 16> end{h.rows, h.part, h.hit, h.parts, h.first_class};
        fp32_gemm_dma_tile<128, 128, 2, 2, false, true, false, false, decltype(end), kFold>(p, blockIdx.x, 0, 4, end);
    } else if constexpr (WHAT == HeadTile::kGradLogits) {
        const GradLogitsEnd<float, 4> end{h.rows, static_cast<float*>(h.d), h.ldd, (h.n + 3) & ~3, h.first_class};
        fp32_gemm_dma_tile<128, 128, 2, 2, false, true, false, false, decltype(end), kFold>(p, blockIdx.x, 0, 4, end);
    } else if constexpr (WHAT == HeadTile::kGradHidden) {
        const int first = blockIdx.z * h.k_chunk;
        p.a += first;
        p.b += first * h.ldb;
        p.k = max(0, min(h.k_chunk, h.k - first));
        p.d += blockIdx.z * h.slice;
        if (h.add) p.c = p.d;
        fp32_gemm_dma_tile<128, 128, 2, 2, false, false, false, false, StoreTile, kFold>(p, blockIdx.x, 0);
    } else {
        const GradWeightEnd end{static_cast<float*>(h.d), h.ldd};
        fp32_gemm_dma_tile<128, 128, 2, 2, false, false, true, false, decltype(end), kFold>(p, blockIdx.x, 0, 4, end, h.read_m, h.read_n);
    }
}

inline dim3 headGrid(const HeadTileArgs& a, int size, int slices) {
    const int64_t tiles = (static_cast<int64_t>(a.m) + size - 1) / size * ((static_cast<int64_t>(a.n) + size - 1) / size);
    if (tiles > INT32_MAX) raise(FTRAIN_STATUS_UNSUPPORTED, "cross entropy: too many tiles (%lld)", (long long)tiles);
    return dim3(static_cast<uint32_t>(tiles), 1, static_cast<uint32_t>(slices));
}

template <bool BF16>
void launchHeadTileHalf(HeadTile what, const HeadTileArgs& args, int slices, hipStream_t stream) {
    const dim3 grid = headGrid(args, 256, slices);
    switch (what) {
        case HeadTile::kLogSum:
            launch(&headTileHalf<BF16, HeadTile::kLogSum>, "cross entropy logits", grid, dim3(512), stream, args);
            break;
        case HeadTile::kGradLogits:
            launch(&headTileHalf<BF16, HeadTile::kGradLogits>, "cross entropy logits' gradient", grid, dim3(512), stream, args);
            break;
        case HeadTile::kGradHidden:
            launch(&headTileHalf<BF16, HeadTile::kGradHidden>, "cross entropy hidden gradient", grid, dim3(512), stream, args);
            break;
        case HeadTile::kGradWeight:
            launch(&headTileHalf<BF16, HeadTile::kGradWeight>, "cross entropy weight gradient", grid, dim3(512), stream, args);
            break;
    }
}

}  // namespace ftrain::train
