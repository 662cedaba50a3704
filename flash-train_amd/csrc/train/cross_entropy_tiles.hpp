// The cross entropy's products on the GEMM's tiles, with the ends below in place of d = alpha acc + beta c:
// 16-bit types on 256x256 (gemm/pingpong_tile.hpp), 128x128 and 64x128 (gemm/dma_tile.hpp), fp32 on 128x128 and
// 64x64 (gemm/dma32_tile.hpp).
#pragma once

#include "../gemm/dma32_tile.hpp"
#include "../gemm/dma_tile.hpp"
#include "../gemm/pingpong_tile.hpp"
#include "cross_entropy.hpp"
#include "device.hpp"
#include "ft/train.hpp"

namespace ftrain::train {

// ---- 16-bit operands: the 256x256 tile of gemm/pingpong_tile.hpp.
//
// A lane holds, of row 128 i + 64 wm + 16 u + j16 of the tile, columns 128 j + 32 wn + 16 v + 4 g + r
// (i, j, v < 2, u, r < 4): acc[i][j][u][v][r].
typedef gemm::ppdev::floatx4 TileSums[2][2][4][2];

struct Place {
    int lane, j16, g, wm, wn, wave;
    __device__ __forceinline__ Place()
        : lane(threadIdx.x & 63), j16(lane & 15), g(lane >> 4),
          wm(__builtin_amdgcn_readfirstlane(threadIdx.x >> 8)),
          wn(__builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3)),
          wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {}
    __device__ __forceinline__ int row(int i, int u) const { return 128 * i + 64 * wm + 16 * u + j16; }
    __device__ __forceinline__ int col(int j, int v) const { return 128 * j + 32 * wn + 16 * v + 4 * g; }
};

// Each row's largest logit and sum of exponentials over the tile's classes.  A lane reduces its 16
// logits of a row by itself, four lanes meet by shuffles, four waves in LDS.  Against a turn of the tile
// through LDS, after which 32 lanes hold a row (ten shuffles for every two rows of a wave): 8192 x 4096 x
// 65536 bf16 3156 -> 2838 us.
struct LogSumEnd16 {
    const RowInfo* rows;
    float2* part;
    float* hit;
    int64_t tokens;
    int M, N, first_class;

    __device__ __forceinline__ void operator()(TileSums& acc, char* lds, int m0, int n0) const {
        const Place at;
        const int rows_left = M - m0, cols_left = N - n0;
        if (cols_left < 256) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (at.col(j, v) + r >= cols_left) {
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int u = 0; u < 4; ++u) acc[i][j][u][v][r] = -INFINITY;
                        }
        }
        float2* const met = reinterpret_cast<float2*>(lds);  // [4][256]
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (128 * i >= rows_left) break;
            int target[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int row = at.row(i, u);
                target[u]     = row < rows_left ? rows[m0 + row].target - first_class - n0 : -1;
            }
            float top[4], sum[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                top[u] = acc[i][0][u][0][0];
#pragma unroll
                for (int q = 1; q < 16; ++q) top[u] = fmaxf(top[u], acc[i][q >> 3][u][(q >> 2) & 1][q & 3]);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) top[u] = fmaxf(top[u], __shfl_xor(top[u], 16, kWave));
#pragma unroll
            for (int u = 0; u < 4; ++u) top[u] = fmaxf(top[u], __shfl_xor(top[u], 32, kWave));
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                // Nothing but minus infinity: the exponentials of the differences would be NaN.
                const float base = top[u] == -INFINITY ? 0.f : top[u];
                sum[u]           = 0.f;
#pragma unroll
                for (int q = 0; q < 16; ++q) sum[u] += expFast(acc[i][q >> 3][u][(q >> 2) & 1][q & 3] - base);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) sum[u] += __shfl_xor(sum[u], 16, kWave);
#pragma unroll
            for (int u = 0; u < 4; ++u) sum[u] += __shfl_xor(sum[u], 32, kWave);
            if (at.g == 0) {
#pragma unroll
                for (int u = 0; u < 4; ++u) met[256 * at.wn + at.row(i, u)] = make_float2(top[u], sum[u]);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int t   = target[u];
                const bool my = t >= 0 && t < min(256, cols_left) && ((t >> 5) & 3) == at.wn && ((t >> 2) & 3) == at.g;
                if (__any(my)) {
                    float x = 0.f;
#pragma unroll
                    for (int q = 0; q < 16; ++q)
                        if ((t >> 7) == (q >> 3) && ((t >> 4) & 1) == ((q >> 2) & 1) && (t & 3) == (q & 3))
                            x = acc[i][q >> 3][u][(q >> 2) & 1][q & 3];
                    if (my) hit[m0 + at.row(i, u)] = x;
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int row = threadIdx.x;
        if (row < 256 && row < rows_left) {
            float2 s[4];
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                s[w] = met[256 * w + row];
                top  = fmaxf(top, s[w].x);
            }
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < 4; ++w) sum += s[w].y * expFast(s[w].x - base);
            part[static_cast<int64_t>((first_class + n0) >> 8) * tokens + m0 + row] = make_float2(top, sum);
        }
    }
};

// dl in the operands' type: g (exp(l - lse) - [the target]), zeros in the padding past the classes.
// Formed where the MFMAs leave it, then turned through LDS (512 bytes a row, 16-byte chunk c of row r at
// slot c ^ (r & 15): no bank conflicts) so that a store covers two rows of 512 bytes.
template <bool BF16>
struct GradLogitsEnd16 {
    using T = std::conditional_t<BF16, bf16, fp16>;
    const RowInfo* rows;
    T* d;
    int64_t ldd;
    int M, N, padded, first_class;

    __device__ __forceinline__ void operator()(TileSums& acc, char* lds, int m0, int n0) const {
        typedef gemm::ppdev::u32x4 u32x4;
        typedef gemm::ppdev::u32x2 u32x2;
        typedef gemm::ppdev::floatx4 floatx4;
        const Place at;
        const int rows_left = M - m0, cols_left = N - n0;
        RowInfo info[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) info[i][u] = rows[m0 + min(at.row(i, u), rows_left - 1)];
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        auto value = [&](floatx4& x, int i, int u, int c, bool last) {
            const RowInfo& r = info[i][u];
            // exp(l - lse) as 2^(l log2 e - lse log2 e): the rounding of the second product, 2^-24 of it,
            // is far below that of the result to 16 bits.
            const float low = r.lse * -kLog2e, g = r.target < 0 ? NAN : r.grad;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], kLog2e, low)) * g;
            if (last) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e >= cols_left) x[e] = 0.f;
            }
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (128 * i >= rows_left) break;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const RowInfo& r = info[i][u];
                if (cols_left >= 256) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) value(acc[i][q >> 1][u][q & 1], i, u, at.col(q >> 1, q & 1), false);
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) value(acc[i][q >> 1][u][q & 1], i, u, at.col(q >> 1, q & 1), true);
                }
                // The target's class, in the few tiles that hold it (a NaN stays one).
                const int y   = r.target - first_class - n0;
                const bool my = y >= 0 && y < min(256, cols_left) && ((y >> 5) & 3) == at.wn && ((y >> 2) & 3) == at.g;
                if (__any(my)) {
#pragma unroll
                    for (int q = 0; q < 16; ++q)
                        if (my && (y >> 7) == (q >> 3) && ((y >> 4) & 1) == ((q >> 2) & 1) && (y & 3) == (q & 3))
                            acc[i][q >> 3][u][(q >> 2) & 1][q & 3] -= r.grad;
                }
                char* const to = lds + at.row(i, u) * 512;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const int c      = at.col(j, v);
                        const floatx4& x = acc[i][j][u][v];
                        *reinterpret_cast<u32x2*>(to + 16 * ((c >> 3) ^ at.j16) + 8 * (at.g & 1)) =
                            u32x2{gemm::ppdev::pack2<BF16>(x[0], x[1]), gemm::ppdev::pack2<BF16>(x[2], x[3])};
                    }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int er = at.lane >> 5, ec = 8 * (at.lane & 31);
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const int row = 32 * at.wave + 2 * t + er;
            if (row < rows_left && n0 + ec < padded)
                *reinterpret_cast<u32x4*>(d + (m0 + row) * ldd + n0 + ec) =
                    *reinterpret_cast<const u32x4*>(lds + row * 512 + 16 * ((ec >> 3) ^ (row & 15)));
        }
    }
};

// ---- 16-bit operands: the 128x128 and 64x128 tiles of gemm/dma_tile.hpp.
//
// Lane (li = lane % 32, h = lane / 32) of wave w holds rows BM / 2 (w / 2) + 32 bi + 8 (r / 4) + 4 h +
// r % 4, column 64 (w % 2) + 32 bj + li: acc[bi][bj][r].  Both ends turn the tile through LDS (512 bytes
// a row; the row's halves change places where bit 2 of the row is set, so the two h write to different
// banks), after which 16 lanes hold 8 adjacent columns each of a row and a wave four rows.
template <int BM>
using TileSums128 = gemm::ddev::floatx16[BM / 64][2];
// Steps of a wave over its rows.
template <int BM>
constexpr int kTurns = BM / 16;

__device__ __forceinline__ int turnedRow(int bm, int t) { return bm / 4 * (threadIdx.x >> 6) + 4 * t + ((threadIdx.x & 63) >> 4); }

// f(t, row, column, v[8]) for the steps t of every wave, rows and columns within the tile.
template <int BM, class F>
__device__ __forceinline__ void turned128(TileSums128<BM>& acc, char* a, char* b, F&& f) {
    typedef gemm::ppdev::floatx4 floatx4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // 64 rows in b's LDS; of 128, rows 0 .. 63, which waves 0 and 1 hold and read again, in a's.
    char* const lds = BM == 64 ? b : wave < 2 ? a : b - 64 * 512;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int bi = 0; bi < BM / 64; ++bi)
#pragma unroll
        for (int bj = 0; bj < 2; ++bj)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = BM / 2 * (wave >> 1) + 32 * bi + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
                const int col = 64 * (wave & 1) + 32 * bj + (lane & 31);
                *reinterpret_cast<float*>(lds + row * 512 + 4 * (col ^ (8 * (row & 4)))) = acc[bi][bj][r];
            }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int t = 0; t < kTurns<BM>; ++t) {
        const int row = turnedRow(BM, t), col = 8 * (lane & 15);
        float v[8];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const floatx4 x = *reinterpret_cast<const floatx4*>(lds + row * 512 + 4 * ((col + 4 * q) ^ (8 * (row & 4))));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * q + e] = x[e];
        }
        f(t, row, col, v);
    }
}

template <int BM>
struct LogSumEnd128 {
    Targets targets;
    float2* part;
    float* hit;
    int64_t tokens;
    int M, N, first_class;

    __device__ __forceinline__ void operator()(TileSums128<BM>& acc, char* a, char* b, int m0, int n0) const {
        const int rows_left = M - m0, cols_left = N - n0;
        int target[kTurns<BM>];
#pragma unroll
        for (int t = 0; t < kTurns<BM>; ++t)
            target[t] = targets(m0 + min(turnedRow(BM, t), rows_left - 1)) - first_class - n0;
        turned128<BM>(acc, a, b, [&](int t, int row, int col, float (&v)[8]) {
            float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (col + e >= cols_left) v[e] = -INFINITY;
                if (col + e == target[t]) x = v[e];
                top = fmaxf(top, v[e]);
            }
            top              = groupMax<16>(top);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += expFast(v[e] - base);
            sum = groupSum<16>(sum);
            if (row >= rows_left) return;
            if (target[t] >= col && target[t] < min(col + 8, cols_left)) hit[m0 + row] = x;
            if (col == 0) part[static_cast<int64_t>((first_class + n0) >> 7) * tokens + m0 + row] = make_float2(top, sum);
        });
    }
};

template <bool BF16, int BM>
struct GradLogitsEnd128 {
    using T = std::conditional_t<BF16, bf16, fp16>;
    const RowInfo* rows;
    T* d;
    int64_t ldd;
    int M, N, padded, first_class, pair;

    __device__ __forceinline__ void operator()(TileSums128<BM>& acc, char* a, char* b, int m0, int n0) const {
        using gemm::ppdev::pack2;
        const int rows_left = M - m0, cols_left = N - n0;
        RowInfo info[kTurns<BM>];
#pragma unroll
        for (int t = 0; t < kTurns<BM>; ++t) info[t] = rows[m0 + min(turnedRow(BM, t), rows_left - 1)];
        turned128<BM>(acc, a, b, [&](int t, int row, int col, float (&v)[8]) {
            const RowInfo r = info[t];
            const int y     = r.target - first_class - n0;
            const float g   = r.target < 0 ? NAN : r.grad;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = (expFast(v[e] - r.lse) - (col + e == y ? 1.f : 0.f)) * g;
                if (col + e >= cols_left) v[e] = 0.f;
            }
            if (row >= rows_left || n0 + col >= padded) return;
            // One or two rows a token (kFewTokens).
            T* const to = d + (m0 + row) * pair * ldd + n0 + col;
            auto store  = [&](T* at) {
                *reinterpret_cast<gemm::ppdev::u32x4*>(at) = gemm::ppdev::u32x4{
                    pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]), pack2<BF16>(v[4], v[5]), pack2<BF16>(v[6], v[7])};
            };
            store(to);
            if (pair == 2) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] -= toFloat(static_cast<T>(v[e]));
                store(to + ldd);
            }
        });
    }
};

// 16-bit dw: rows of any address.  (The tile's own end stores 2 bytes a lane.)
template <bool BF16>
struct GradWeightEnd128 {
    using T = std::conditional_t<BF16, bf16, fp16>;
    T* d;
    int64_t ldd;
    int M, N;
    float alpha;

    __device__ __forceinline__ void operator()(TileSums128<128>& acc, char* a, char* b, int m0, int n0) const {
        const int rows_left = M - m0, cols_left = N - n0;
        turned128<128>(acc, a, b, [&](int, int row, int col, float (&v)[8]) {
            if (row >= rows_left || col >= cols_left) return;
            T* const to = d + (m0 + row) * ldd + n0 + col;
            Pack<T> out;
#pragma unroll
            for (int e = 0; e < 8; ++e) out.v[e] = static_cast<T>(v[e] * alpha);
            if (col + 8 <= cols_left) {
                *reinterpret_cast<Pack<T>*>(to) = out;
            } else {
#pragma unroll
                for (int e = 0; e < 7; ++e)
                    if (col + e < cols_left) to[e] = out.v[e];
            }
        });
    }
};

// ---- fp32: the tiles of gemm/dma32_tile.hpp, four adjacent sums of a row at a time.

// A row's largest logit and sum of exponentials over the 64 classes that 16 lanes hold.
struct LogSumEnd32 {
    Targets targets;
    float2* part;
    float* hit;
    int64_t tokens;
    int first_class;

    __device__ __forceinline__ void operator()(int row, int col, float (&v)[4], bool inside, int left) const {
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (e >= left) v[e] = -INFINITY;
            top = fmaxf(top, v[e]);
        }
        top              = groupMax<16>(top);
        const float base = top == -INFINITY ? 0.f : top;
        float sum        = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += expFast(v[e] - base);
        sum = groupSum<16>(sum);
        if (!inside) return;
        const int at = targets(row) - first_class - col;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e == at && e < left) hit[row] = v[e];
        // (The lanes' classes may all lie past the last.)
        if (threadIdx.x % 16 == 0 && left > 0)
            part[static_cast<int64_t>((first_class + col) >> 6) * tokens + row] = make_float2(top, sum);
    }
};

struct GradLogitsEnd32 {
    const RowInfo* rows;
    float* d;
    int64_t ldd;
    int padded, first_class;

    __device__ __forceinline__ void operator()(int row, int col, float (&v)[4], bool inside, int left) const {
        if (!inside || col >= padded) return;
        const RowInfo r = rows[row];
        const int at    = r.target - first_class - col;
        const float g   = r.target < 0 ? NAN : r.grad;
        float4 out;
        float* const o = &out.x;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = e < left ? (expFast(v[e] - r.lse) - (e == at ? 1.f : 0.f)) * g : 0.f;
        *reinterpret_cast<float4*>(d + row * ldd + col) = out;
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
__device__ __forceinline__ bool tileProblem(const HeadTileArgs& h, P& p, int size, int tile_cols, int tile) {
    constexpr bool kOfDl = WHAT == HeadTile::kGradHidden || WHAT == HeadTile::kGradWeight;
    const int valid      = h.head == nullptr ? h.m : h.head->valid * (kOfDl ? h.pair : 1);
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
    return tile < p.tiles_m * p.tiles_n;
}

template <bool BF16, HeadTile WHAT>
__global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2))) void headTileHalf(HeadTileArgs h) {
    using T = std::conditional_t<BF16, bf16, fp16>;
    gemm::HalfGemmParams p{};
    if (!tileProblem<WHAT>(h, p, 256, 256, blockIdx.x)) return;
    p.a = h.a, p.b = h.b, p.d = h.d;
    using gemm::ppdev::half_gemm_pp_tile;
    using gemm::ppdev::kBand;
    if constexpr (WHAT == HeadTile::kLogSum) {
        half_gemm_pp_tile<BF16, false, true>(p, blockIdx.x, kBand,
                                             LogSumEnd16{h.targets.rows, h.part, h.hit, h.tokens, p.m, p.n, h.first_class});
    } else if constexpr (WHAT == HeadTile::kGradLogits) {
        half_gemm_pp_tile<BF16, false, true>(
            p, blockIdx.x, kBand,
            GradLogitsEnd16<BF16>{h.targets.rows, static_cast<T*>(h.d), h.ldd, p.m, p.n, (h.n + 7) & ~7, h.first_class});
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

// Tile `tile` of slice z of dx, with NB stage buffers.
template <bool BF16, int BM, int NB>
__device__ __forceinline__ void gradHiddenTile(const HeadTileArgs& h, int tile, int z) {
    using T = std::conditional_t<BF16, bf16, fp16>;
    gemm::HalfGemmParams p{};
    if (!tileProblem<HeadTile::kGradHidden>(h, p, BM, 128, tile)) return;
    const int first = z * h.k_chunk;
    p.a             = static_cast<const T*>(h.a) + first;
    p.b             = static_cast<const T*>(h.b) + first * h.ldb;
    p.k             = max(0, min(h.k_chunk, h.k - first));
    p.d             = static_cast<float*>(h.d) + z * h.slice;
    if (h.add) p.c = p.d;
    gemm::ddev::half_gemm_dma_tile<BF16, false, false, 128, false, BM, NB>(p, tile);
}

// Tile `tile` of dw.  Two stage buffers, two workgroups to a CU: k, the tokens, is short.
template <bool BF16>
__device__ __forceinline__ void gradWeightTile(const HeadTileArgs& h, int tile) {
    using T   = std::conditional_t<BF16, bf16, fp16>;
    using End = GradWeightEnd128<BF16>;
    gemm::HalfGemmParams p{};
    if (!tileProblem<HeadTile::kGradWeight>(h, p, 128, 128, tile)) return;
    p.a = h.a, p.b = h.b;
    gemm::ddev::half_gemm_dma_tile<BF16, true, false, 128, false, 128, 2, false, End>(
        p, tile, 0, 8, End{static_cast<T*>(h.d), h.ldd, p.m, p.n, h.head->inv_scale}, h.read_m, h.read_n);
}

// BM 128: three stage buffers, as this tile runs where there are few workgroups to a CU (one needs two
// stages in flight to be busy by itself).  BM 64, two on a CU, for at most 64 tokens, whose products are
// the weight's reading (16 x 4096 x 32003 bf16 loss, 262 MB, 76 -> 58 us), and for the logits of few tiles.
// ROTATE: neighbouring column tiles start at different stages, or all workgroups would read the same few
// HBM channels at once where the weight's rows are a power of two apart.
template <bool BF16, HeadTile WHAT, int BM>
__global__ __launch_bounds__(256, BM == 64 || WHAT == HeadTile::kGradWeight ? 2 : 1) void headTileHalf128(HeadTileArgs h) {
    using T = std::conditional_t<BF16, bf16, fp16>;
    using gemm::ddev::half_gemm_dma_tile;
    if constexpr (WHAT == HeadTile::kGradHidden) {
        gradHiddenTile<BF16, BM, 3>(h, blockIdx.x, blockIdx.z);
    } else if constexpr (WHAT == HeadTile::kGradWeight) {
        gradWeightTile<BF16>(h, blockIdx.x);
    } else {
        gemm::HalfGemmParams p{};
        if (!tileProblem<WHAT>(h, p, BM, 128, blockIdx.x)) return;
        p.a = h.a, p.b = h.b, p.d = h.d;
        if constexpr (WHAT == HeadTile::kLogSum) {
            using End = LogSumEnd128<BM>;
            half_gemm_dma_tile<BF16, false, true, 128, false, BM, 3, true, End>(
                p, blockIdx.x, 0, 8, End{h.targets, h.part, h.hit, h.tokens, p.m, p.n, h.first_class});
        } else if constexpr (WHAT == HeadTile::kGradLogits) {
            using End = GradLogitsEnd128<BF16, BM>;
            half_gemm_dma_tile<BF16, false, true, 128, false, BM, 3, true, End>(
                p, blockIdx.x, 0, 8, End{h.targets.rows, static_cast<T*>(h.d), h.ldd, p.m, p.n, (h.n + 7) & ~7, h.first_class, h.pair});
        } else {
            const int first = blockIdx.z * h.k_chunk;
            p.a             = static_cast<const T*>(h.a) + first;
            p.b             = static_cast<const T*>(h.b) + first;
            p.k             = max(0, min(h.k_chunk, h.k - first));
            p.d             = static_cast<float*>(h.d) + blockIdx.z * h.slice;
            half_gemm_dma_tile<BF16, false, true, 128, false, BM, 3, true>(p, blockIdx.x);
        }
    }
}

// dx's slices, `tiles` workgroups each, then dw's tiles: one launch for the two products of dl where both
// are on this tile.
template <bool BF16>
__global__ __launch_bounds__(256, 2) void headGradients(HeadTileArgs hidden, HeadTileArgs weight, int tiles, int slices) {
    const int at = static_cast<int>(blockIdx.x) - tiles * slices;
    if (at < 0)
        gradHiddenTile<BF16, 128, 2>(hidden, blockIdx.x % tiles, blockIdx.x / tiles);
    else
        gradWeightTile<BF16>(weight, at);
}

// The logits' sums of k: on the 64x64 tile those of every 256 apart and then added up, as a loss near 0 is as
// exact as its logits.  Root mean square errors of losses near 10, in one chain / so: 16 x 8192 x 20000 7.2e-6 /
// 6.1e-7, 16 x 1000 x 1000 1.7e-6 / 6.3e-7, 100 x 8192 x 1000 4.7e-6 / 5.7e-7; of dl's products, of their size,
// 16 x 8192 x 20000 1.2e-5 / 1.5e-6, 100 x 4096 x 1000 1.5e-5 / 1.3e-6.  dl of more tokens than kApartTokens, whose
// errors are many, and the 128x128 tile: one chain, as in the GEMM itself (5e-6 of dl's size at k = 2048, 1.5e-5
// at 8192), which the results then agree with; on the large tile it took 5% more time (16 accumulators' worth of
// spills at 256 registers).
template <HeadTile WHAT, int BM>
__global__ __launch_bounds__(256, 2) void headTileFp32(HeadTileArgs h) {
    constexpr int WM = BM == 128 ? 2 : 4, WN = BM == 128 ? 2 : 1;
    gemm::GemmParams p{};
    if (!tileProblem<WHAT>(h, p, BM, BM, blockIdx.x)) return;
    p.a = static_cast<const float*>(h.a), p.b = static_cast<const float*>(h.b), p.d = static_cast<float*>(h.d);
    using gemm::d32::fp32_gemm_dma_tile;
    using gemm::d32::StoreTile;
    constexpr int kFold = BM == 64 ? 8 : 0;  // stages
    if constexpr (WHAT == HeadTile::kLogSum) {
        using End = LogSumEnd32;
        fp32_gemm_dma_tile<BM, BM, WM, WN, false, true, false, false, End, kFold>(
            p, blockIdx.x, 0, 4, End{h.targets, h.part, h.hit, h.tokens, h.first_class});
    } else if constexpr (WHAT == HeadTile::kGradLogits) {
        using End = GradLogitsEnd32;
        fp32_gemm_dma_tile<BM, BM, WM, WN, false, true, false, false, End, kFold>(
            p, blockIdx.x, 0, 4, End{h.targets.rows, static_cast<float*>(h.d), h.ldd, (h.n + 3) & ~3, h.first_class}, 0, 0, h.m <= kApartTokens);
    } else if constexpr (WHAT == HeadTile::kGradHidden) {
        const int first = blockIdx.z * h.k_chunk;
        p.a += first;
        p.b += first * h.ldb;
        p.k = max(0, min(h.k_chunk, h.k - first));
        p.d += blockIdx.z * h.slice;
        if (h.add) p.c = p.d;
        fp32_gemm_dma_tile<BM, BM, WM, WN, false, false, false, false, StoreTile>(p, blockIdx.x, 0);
    } else if constexpr (WHAT == HeadTile::kLogits) {
        const int first = blockIdx.z * h.k_chunk;
        p.a += first;
        p.b += first;
        p.k = max(0, min(h.k_chunk, h.k - first));
        p.d += blockIdx.z * h.slice;
        // Whole chunks of four columns are stored; the row stride has room for them.
        p.n = (h.n + 3) & ~3;
        fp32_gemm_dma_tile<BM, BM, WM, WN, false, true, false, false, StoreTile, kFold>(p, blockIdx.x, 0, 4, StoreTile{}, 0, h.n);
    } else {
        using End = GradWeightEnd;
        fp32_gemm_dma_tile<BM, BM, WM, WN, false, false, true, false, End>(
            p, blockIdx.x, 0, 4, End{static_cast<float*>(h.d), h.ldd}, h.read_m, h.read_n);
    }
}

inline uint32_t headTiles(const HeadTileArgs& a, int rows, int cols) {
    const int64_t tiles = (static_cast<int64_t>(a.m) + rows - 1) / rows * ((static_cast<int64_t>(a.n) + cols - 1) / cols);
    if (tiles > INT32_MAX / 2) raise(FTRAIN_STATUS_UNSUPPORTED, "cross entropy: too many tiles (%lld)", (long long)tiles);
    return static_cast<uint32_t>(tiles);
}

template <class K>
void launchHead(K kernel, const char* name, const HeadTileArgs& a, int rows, int cols, int threads, int slices,
                hipStream_t stream) {
    launch(kernel, name, dim3(headTiles(a, rows, cols), 1, static_cast<uint32_t>(slices)), dim3(threads), stream, a);
}

constexpr const char* kHeadNames[5] = {"cross entropy loss", "cross entropy logits' gradient", "cross entropy hidden gradient",
                                       "cross entropy weight gradient", "cross entropy logits"};

template <bool BF16>
void launchHeadTileHalf(HeadTile what, int rows, const HeadTileArgs& args, int slices, hipStream_t stream) {
    using W = HeadTile;
    constexpr void (*large[4])(HeadTileArgs) = {&headTileHalf<BF16, W::kLogSum>, &headTileHalf<BF16, W::kGradLogits>,
                                                &headTileHalf<BF16, W::kGradHidden>, &headTileHalf<BF16, W::kGradWeight>};
    constexpr void (*medium[5])(HeadTileArgs) = {
        &headTileHalf128<BF16, W::kLogSum, 128>, &headTileHalf128<BF16, W::kGradLogits, 128>, &headTileHalf128<BF16, W::kGradHidden, 128>,
        &headTileHalf128<BF16, W::kGradWeight, 128>, &headTileHalf128<BF16, W::kLogits, 128>};
    constexpr void (*small[5])(HeadTileArgs) = {&headTileHalf128<BF16, W::kLogSum, 64>, &headTileHalf128<BF16, W::kGradLogits, 64>,
                                                &headTileHalf128<BF16, W::kGradHidden, 64>, nullptr,
                                                &headTileHalf128<BF16, W::kLogits, 64>};
    const int i = static_cast<int>(what);
    if (rows == 256)
        launchHead(large[i], kHeadNames[i], args, 256, 256, 512, slices, stream);
    else
        launchHead(rows == 128 ? medium[i] : small[i], kHeadNames[i], args, rows, 128, 256, slices, stream);
}

template <bool BF16>
void launchHeadGradientsHalf(const HeadTileArgs& hidden, int slices, const HeadTileArgs& weight, hipStream_t stream) {
    const uint32_t tiles = headTiles(hidden, 128, 128);
    launch(&headGradients<BF16>, "cross entropy gradients", dim3(tiles * slices + headTiles(weight, 128, 128)), dim3(256), stream,
           hidden, weight, static_cast<int>(tiles), slices);
}

}  // namespace ftrain::train
