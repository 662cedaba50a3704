// The router of a mixture of experts.  For each row t of the logits l (tokens x experts):
//   p_t = softmax(l_t); the top_k experts by logit, ties to the lowest index; their gates p (or p
//   over the sum of the chosen p); the packed row ("slot") of each choice when the choices are
//   ordered by expert, then by token, then by rank; counts_e, the choices of expert e; and
//   loss = E sum_e f_e P_e, f_e = counts_e / sum counts, P_e the mean of p_te over the routed rows.
// A row that the mask drops, or with every logit minus infinity, is not routed: its experts and slots
// are -1, its gates 0, and it counts nowhere.  A logit of minus infinity is never chosen, nor is a NaN.
// Backward, the counts taken as constants:
//   dp_te = gl E f_e / N + [e chosen] dgate, dl_t = p_t (dp_t - sum_e p_te dp_te)
// and with normalised gates w the chosen entries' part is w (dgate - sum w dgate) instead.
//
// A group of G lanes owns a row, eight logits in each lane (16 above 512 experts): softmax and
// selection stay in registers and cross the group by lane shuffles.  A workgroup takes a run of
// consecutive rows, so the order of the choices within an expert is the order of (workgroup, row,
// rank): `choose` counts each workgroup's choices, `scan` turns them into each workgroup's first
// rank (one workgroup per expert), `place` hands out the slots.  Sums over rows are taken in a fixed
// order; the only atomics count in LDS, in whole numbers.
#include <algorithm>

#include "device.hpp"
#include "ft/train.hpp"

namespace ftrain::train {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves   = kThreads / kWave;
// Most workgroups: four on each of the 256 CUs.
constexpr int kMaxBlocks = 1024;

struct RouteArgs {
    const void* logits;
    const uint8_t* mask;
    int32_t *experts, *slots, *counts, *routed;
    float *gates, *loss;
    const float *grad_gates, *grad_loss;
    void* grad_logits;
    int64_t rows, ld, grad_ld;
    int32_t n_experts, top_k, rows_per_block, blocks;
    int32_t normalize;
    // Workspace: of each expert, each workgroup's choices (then their first rank) and sum of p; of
    // each workgroup, its routed rows; of each expert, its sum of p.
    int32_t* block_count;
    float* block_p;
    int32_t* block_routed;
    float* sum_p;
};

// A row's logits in registers: lane g of the group's G lanes holds VPL of them.  VEC: adjacent ones
// (16-byte loads), else every G-th one (adjacent lanes load adjacent logits).
template <class T, int VPL, int G, bool VEC>
struct Row {
    float v[VPL];
    int g;

    __device__ __forceinline__ int index(int j) const { return VEC ? g * VPL + j : g + G * j; }
    __device__ __forceinline__ void load(const T* row, int n) {
        if constexpr (VEC) {
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < VPL; j += N) {
                if (index(j) < n) {
                    typedef T vec __attribute__((ext_vector_type(N)));
                    const vec x = *reinterpret_cast<const vec*>(row + index(j));
#pragma unroll
                    for (int e = 0; e < N; ++e) v[j + e] = toFloat(static_cast<T>(x[e]));
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) v[j + e] = -INFINITY;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j) v[j] = index(j) < n ? toFloat(row[index(j)]) : -INFINITY;
        }
    }
    // Exponentials relative to the largest logit into p; their sum is returned.  any: some logit is
    // not minus infinity.
    __device__ __forceinline__ float exponentials(float (&p)[VPL], float& top, bool& any) const {
        float m = -INFINITY;
        int some = 0;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            m = fmaxf(m, v[j]);
            some |= v[j] != -INFINITY;
        }
        top = groupMax<G>(m);
#pragma unroll
        for (int d = 1; d < G; d <<= 1) some |= __shfl_xor(some, d, kWave);
        any         = some != 0;
        float total = 0.f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            p[j] = expf(v[j] - top);
            total += p[j];
        }
        return groupSum<G>(total);
    }
};

template <class T, int VPL, int G, bool VEC>
__global__ __launch_bounds__(kThreads) void choose(RouteArgs a) {
    constexpr int kRows = kThreads / G;  // rows at a time
    __shared__ int hist[kMaxExperts];
    __shared__ float sums[kThreads * VPL];
    __shared__ int routed_of[kRows];
    const int group = threadIdx.x / G, n = a.n_experts;
    Row<T, VPL, G, VEC> row;
    row.g = threadIdx.x % G;
    for (int e = threadIdx.x; e < n; e += kThreads) hist[e] = 0;
    __syncthreads();

    float sum_p[VPL] = {};
    int routed       = 0;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.rows_per_block;
    const int64_t last  = min(first + a.rows_per_block, a.rows);
    for (int64_t t = first + group; t < last; t += kRows) {
        const bool kept = a.mask == nullptr || a.mask[t] != 0;
        int32_t* const experts = a.experts + t * a.top_k;
        float* const gates     = a.gates + t * a.top_k;
        float p[VPL], top = 0.f, total = 1.f;
        bool any = false;
        if (kept) {
            row.load(static_cast<const T*>(a.logits) + t * a.ld, n);
            total = row.exponentials(p, top, any);
        }
        if (!any) {
            for (int k = row.g; k < a.top_k; k += G) {
                experts[k] = -1;
                gates[k]   = 0.f;
            }
            continue;
        }
        const float inv = 1.f / total;
#pragma unroll
        for (int j = 0; j < VPL; ++j) sum_p[j] += row.index(j) < n ? p[j] * inv : 0.f;
        ++routed;
        float chosen = 0.f;  // sum of the chosen p
        float gate   = 0.f;  // lane k % G keeps the gates k, k + G ..: written at once below
        for (int k = 0; k < a.top_k; ++k) {
            float best = -INFINITY;
            int at     = n;
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (row.v[j] > best) best = row.v[j], at = row.index(j);
#pragma unroll
            for (int d = 1; d < G; d <<= 1) {
                const float other = __shfl_xor(best, d, kWave);
                const int oat     = __shfl_xor(at, d, kWave);
                if (other > best || (other == best && oat < at)) best = other, at = oat;
            }
            const bool found = at < n;
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (row.index(j) == at) row.v[j] = -INFINITY;
            // A row whose sum is NaN has NaN gates.
            gate = found ? expf(best - top) * inv : 0.f;
            chosen += gate;
            if (row.g == 0) {
                experts[k] = found ? at : -1;
                gates[k]   = gate;
                if (found) atomicAdd(&hist[at], 1);
            }
        }
        if (a.normalize && row.g == 0)
            for (int k = 0; k < a.top_k; ++k) gates[k] = experts[k] >= 0 ? gates[k] / chosen : 0.f;
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) sums[group * (G * VPL) + row.index(j)] = sum_p[j];
    if (row.g == 0) routed_of[group] = routed;
    __syncthreads();
    for (int e = threadIdx.x; e < n; e += kThreads) {
        float s = 0.f;
        for (int r = 0; r < kRows; ++r) s += sums[r * (G * VPL) + e];
        a.block_count[static_cast<int64_t>(e) * a.blocks + blockIdx.x] = hist[e];
        a.block_p[static_cast<int64_t>(e) * a.blocks + blockIdx.x]     = s;
    }
    if (threadIdx.x == 0) {
        int s = 0;
        for (int r = 0; r < kRows; ++r) s += routed_of[r];
        a.block_routed[blockIdx.x] = s;
    }
}

// Exclusive prefix sum of one value a thread over the workgroup; total: the sum.
__device__ __forceinline__ int blockScan(int v, int& total) {
    __shared__ int wave_sum[kWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int s = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int up = __shfl_up(s, d, kWave);
        if (lane >= d) s += up;
    }
    if (lane == kWave - 1) wave_sum[wave] = s;
    __syncthreads();
    int before = 0;
    total      = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += wave_sum[w];
        total += wave_sum[w];
    }
    __syncthreads();
    return before + s - v;
}

// Expert blockIdx.x: each workgroup's first rank in place of its count, the expert's count, its sum of p.
__global__ __launch_bounds__(kThreads) void scan(RouteArgs a) {
    int32_t* const count = a.block_count + static_cast<int64_t>(blockIdx.x) * a.blocks;
    const float* const p = a.block_p + static_cast<int64_t>(blockIdx.x) * a.blocks;
    __shared__ float part[kWaves];
    int before = 0;
    float sum  = 0.f;
    for (int b0 = 0; b0 < a.blocks; b0 += kThreads) {
        const int b  = b0 + threadIdx.x;
        const bool in = b < a.blocks;
        int total;
        const int at = blockScan(in ? count[b] : 0, total);
        if (in) {
            count[b] = before + at;
            sum += p[b];
        }
        before += total;
    }
    sum = groupSum<kWave>(sum);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWaves; ++w) sum += part[w];
        a.counts[blockIdx.x] = before;
        a.sum_p[blockIdx.x]  = sum;
    }
}

// The slots of the workgroup's choices; workgroup 0 also finishes the loss.
__global__ __launch_bounds__(kThreads) void place(RouteArgs a) {
    __shared__ int first[kMaxExperts];            // slot of the workgroup's first choice of each expert
    __shared__ int next[kWaves][kMaxExperts];     // each wave's choices, then its next slot
    const int n = a.n_experts, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    int before = 0;
    for (int e0 = 0; e0 < n; e0 += kThreads) {
        const int e = e0 + threadIdx.x;
        int total;
        const int at = blockScan(e < n ? a.counts[e] : 0, total);
        if (e < n) first[e] = before + at;
        before += total;
    }
    for (int e = threadIdx.x; e < n; e += kThreads) {
        first[e] += a.block_count[static_cast<int64_t>(e) * a.blocks + blockIdx.x];
        for (int w = 0; w < kWaves; ++w) next[w][e] = 0;
    }
    __syncthreads();
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.rows_per_block * a.top_k;
    const int64_t end   = min(begin + static_cast<int64_t>(a.rows_per_block) * a.top_k, a.rows * a.top_k);
    const int per_wave  = static_cast<int>((end - begin + kThreads - 1) / kThreads) * kWave;
    const int64_t mine = min(begin + static_cast<int64_t>(wave) * per_wave, end), stop = min(mine + per_wave, end);
    for (int64_t i = mine + lane; i < stop; i += kWave) {
        const int e = a.experts[i];
        if (e >= 0) atomicAdd(&next[wave][e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n; e += kThreads) {
        int at = first[e];
        for (int w = 0; w < kWaves; ++w) {
            const int c = next[w][e];
            next[w][e]  = at;
            at += c;
        }
    }
    __syncthreads();
    for (int64_t i0 = mine; i0 < stop; i0 += kWave) {
        const int64_t i = i0 + lane;
        const int e     = i < stop ? a.experts[i] : -1;
        // The lanes with the same expert: agreement in every bit of its index.
        unsigned long long peers = __ballot(e >= 0);
        for (int bit = 1; bit < n; bit <<= 1) {
            const unsigned long long set = __ballot((e & bit) != 0);
            peers &= (e & bit) ? set : ~set;
        }
        int slot = -1;
        if (e >= 0) {
            const int rank = __popcll(peers & ((1ull << lane) - 1ull));
            slot           = next[wave][e] + rank;
        }
        // Every lane has read before the last of each expert's lanes writes, and the next round reads
        // after it: one wave's LDS accesses are done in order.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (e >= 0 && (peers >> lane) == 1ull) next[wave][e] = slot + 1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (i < stop) a.slots[i] = slot;
    }

    if (blockIdx.x != 0) return;
    __shared__ float part[kWaves];
    int routed = 0, total = 0;
    for (int b = threadIdx.x; b < a.blocks; b += kThreads) routed += a.block_routed[b];
    float dot = 0.f;
    for (int e = threadIdx.x; e < n; e += kThreads) {
        total += a.counts[e];
        dot += static_cast<float>(a.counts[e]) * a.sum_p[e];
    }
    int all_routed, all;
    (void)blockScan(routed, all_routed);
    (void)blockScan(total, all);
    dot = groupSum<kWave>(dot);
    if (lane == 0) part[wave] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWaves; ++w) dot += part[w];
        *a.routed = all_routed;
        *a.loss   = static_cast<float>(n) * (dot / static_cast<float>(max(all, 1))) / static_cast<float>(max(all_routed, 1));
    }
}

template <class T, int VPL, int G, bool VEC>
__global__ __launch_bounds__(kThreads) void backward(RouteArgs a) {
    constexpr int kRows = kThreads / G;
    const int group = threadIdx.x / G, n = a.n_experts;
    Row<T, VPL, G, VEC> row;
    row.g = threadIdx.x % G;
    int total = 0, all;
    for (int e = threadIdx.x; e < n; e += kThreads) total += a.counts[e];
    (void)blockScan(total, all);
    // d loss / d p_te
    const float factor = *a.grad_loss * static_cast<float>(n) / static_cast<float>(max(all, 1)) /
                         static_cast<float>(max(*a.routed, 1));
    float balance[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j)
        balance[j] = row.index(j) < n ? factor * static_cast<float>(a.counts[row.index(j)]) : 0.f;

    const int64_t stride = static_cast<int64_t>(gridDim.x) * kRows;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * kRows + group; t < a.rows; t += stride) {
        T* const out = static_cast<T*>(a.grad_logits) + t * a.grad_ld;
        float p[VPL], d[VPL], top, inv = 0.f;
        bool any = false;
        if (a.mask == nullptr || a.mask[t] != 0) {
            row.load(static_cast<const T*>(a.logits) + t * a.ld, n);
            inv = 1.f / row.exponentials(p, top, any);
        }
        if (any) {
            const int32_t* const experts = a.experts + t * a.top_k;
            const float* const grads     = a.grad_gates + t * a.top_k;
            float dot = 0.f;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                p[j] = row.index(j) < n ? p[j] * inv : 0.f;
                d[j] = balance[j];
            }
            if (a.normalize) {
                // Of the chosen: sum of p, and sum of p dgate; both over the group.
                float picked = 0.f, weighted = 0.f, dg[VPL] = {};
                unsigned is = 0;
                for (int k = 0; k < a.top_k; ++k) {
                    const int e     = experts[k];
                    const float dgk = grads[k];
#pragma unroll
                    for (int j = 0; j < VPL; ++j)
                        if (row.index(j) == e) {
                            dg[j] = dgk;
                            is |= 1u << j;
                            picked += p[j];
                            weighted += p[j] * dgk;
                        }
                }
                picked   = groupSum<G>(picked);
                weighted = groupSum<G>(weighted);
#pragma unroll
                for (int j = 0; j < VPL; ++j) dot += p[j] * d[j];
                dot = groupSum<G>(dot);
                const float mean = weighted / picked;
#pragma unroll
                for (int j = 0; j < VPL; ++j)
                    d[j] = p[j] * (d[j] - dot) + ((is >> j) & 1u ? p[j] / picked * (dg[j] - mean) : 0.f);
            } else {
                for (int k = 0; k < a.top_k; ++k) {
                    const int e     = experts[k];
                    const float dgk = grads[k];
#pragma unroll
                    for (int j = 0; j < VPL; ++j)
                        if (row.index(j) == e) d[j] += dgk;
                }
#pragma unroll
                for (int j = 0; j < VPL; ++j) dot += p[j] * d[j];
                dot = groupSum<G>(dot);
#pragma unroll
                for (int j = 0; j < VPL; ++j) d[j] = p[j] * (d[j] - dot);
            }
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j) d[j] = 0.f;
        }
        if constexpr (VEC) {
            constexpr int N = 16 / sizeof(T);
            typedef T vec __attribute__((ext_vector_type(N)));
#pragma unroll
            for (int j = 0; j < VPL; j += N) {
                vec x;
#pragma unroll
                for (int e = 0; e < N; ++e) x[e] = static_cast<T>(d[j + e]);
                if (row.index(j) < n) *reinterpret_cast<vec*>(out + row.index(j)) = x;
            }
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (row.index(j) < n) out[row.index(j)] = static_cast<T>(d[j]);
        }
    }
}

using Kernel = void (*)(RouteArgs);

template <class T, bool VEC, bool BACK>
Kernel kernelFor(int n, int& lanes) {
    auto pick = [&](auto g, auto vpl) -> Kernel {
        constexpr int G = decltype(g)::value, VPL = decltype(vpl)::value;
        lanes = G;
        if constexpr (BACK)
            return &backward<T, VPL, G, VEC>;
        else
            return &choose<T, VPL, G, VEC>;
    };
    using std::integral_constant;
    const integral_constant<int, 8> eight;
    if (n <= 8) return pick(integral_constant<int, 1>{}, eight);
    if (n <= 16) return pick(integral_constant<int, 2>{}, eight);
    if (n <= 32) return pick(integral_constant<int, 4>{}, eight);
    if (n <= 64) return pick(integral_constant<int, 8>{}, eight);
    if (n <= 128) return pick(integral_constant<int, 16>{}, eight);
    if (n <= 256) return pick(integral_constant<int, 32>{}, eight);
    if (n <= 512) return pick(integral_constant<int, 64>{}, eight);
    return pick(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

template <bool BACK>
Kernel kernelFor(FTrainNumericType type, bool vec, int n, int& lanes) {
    if (type == FTRAIN_NUMERIC_TYPE_FP32)
        return vec ? kernelFor<float, true, BACK>(n, lanes) : kernelFor<float, false, BACK>(n, lanes);
    if (type == FTRAIN_NUMERIC_TYPE_BF16)
        return vec ? kernelFor<bf16, true, BACK>(n, lanes) : kernelFor<bf16, false, BACK>(n, lanes);
    return vec ? kernelFor<fp16, true, BACK>(n, lanes) : kernelFor<fp16, false, BACK>(n, lanes);
}

// Whether rows take whole 16-byte accesses.
bool vectorRows(const Rows& r, FTrainNumericType type) {
    const int64_t n = 16 / static_cast<int64_t>(elementBytes(type));
    return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.ld % n == 0 && r.cols % n == 0;
}

RouteArgs arguments(const MoeRoute& p) {
    RouteArgs a{};
    a.logits      = p.logits.data;
    a.mask        = p.mask;
    a.experts     = p.experts;
    a.slots       = p.slots;
    a.counts      = p.counts;
    a.routed      = p.routed;
    a.gates       = p.gates;
    a.loss        = p.balance_loss;
    a.grad_gates  = p.grad_gates;
    a.grad_loss   = p.grad_loss;
    a.grad_logits = p.grad_logits.data;
    a.rows        = p.logits.rows;
    a.ld          = p.logits.ld;
    a.grad_ld     = p.grad_logits.ld;
    a.n_experts   = static_cast<int32_t>(p.logits.cols);
    a.top_k       = p.top_k;
    a.normalize   = p.normalize;
    return a;
}

uint64_t ceilDiv(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

}  // namespace

uint64_t moeRouteWorkspace(int64_t, int64_t experts) {
    return (2 * static_cast<uint64_t>(experts) * kMaxBlocks + kMaxBlocks + static_cast<uint64_t>(experts)) * 4;
}

void moeRouteForward(const MoeRoute& p, void* workspace, hipStream_t stream) {
    RouteArgs a = arguments(p);
    int lanes   = 0;
    const Kernel kernel =
        kernelFor<false>(p.type, vectorRows(p.logits, p.type), static_cast<int>(p.logits.cols), lanes);
    // Whole passes of the workgroup, at most kMaxBlocks workgroups.
    const uint64_t at_once = kThreads / lanes;
    const uint64_t passes  = std::max<uint64_t>(1, ceilDiv(ceilDiv(a.rows, at_once), kMaxBlocks));
    a.rows_per_block       = static_cast<int32_t>(passes * at_once);
    a.blocks               = static_cast<int32_t>(std::max<uint64_t>(1, ceilDiv(a.rows, a.rows_per_block)));
    a.block_count          = static_cast<int32_t*>(workspace);
    a.block_p              = reinterpret_cast<float*>(a.block_count + p.logits.cols * kMaxBlocks);
    a.block_routed         = reinterpret_cast<int32_t*>(a.block_p + p.logits.cols * kMaxBlocks);
    a.sum_p                = reinterpret_cast<float*>(a.block_routed + kMaxBlocks);
    launch(kernel, "router choose", dim3(a.blocks), dim3(kThreads), stream, a);
    launch(&scan, "router scan", dim3(a.n_experts), dim3(kThreads), stream, a);
    launch(&place, "router place", dim3(a.blocks), dim3(kThreads), stream, a);
}

void moeRouteBackward(const MoeRoute& p, hipStream_t stream) {
    RouteArgs a = arguments(p);
    if (a.rows == 0) return;
    int lanes = 0;
    const bool vec = vectorRows(p.logits, p.type) && vectorRows(p.grad_logits, p.type);
    const Kernel kernel    = kernelFor<true>(p.type, vec, static_cast<int>(p.logits.cols), lanes);
    const uint64_t at_once = kThreads / lanes;
    launch(kernel, "router backward", dim3(static_cast<uint32_t>(std::min<uint64_t>(ceilDiv(a.rows, at_once), 2 * kMaxBlocks))),
           dim3(kThreads), stream, a);
}

}  // namespace ftrain::train
