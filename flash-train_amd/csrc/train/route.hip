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
// A group of G lanes owns a row, eight logits in each lane (16 above 128 experts): softmax and selection
// stay in registers and cross the group by lane permutations.  With many experts vector instructions
// bound the choice, 131072 x 256 fp32, top 8: pairs of value and index reduced by shuffles 148 us,
// maxima first and then the place by a ballot 109, on whole numbers 87 (eight a lane), 59 (16 a lane: the
// steps across lanes serve four rows of a wave instead of two), 55 with the numbers in LDS, 44 with the
// next row's loads under way and the numbers in 16-byte writes to different banks (3.0 TB/s; the reads
// alone would be 27 us).  A workgroup takes a run of consecutive rows, so the order of the choices within
// an expert is the order of (workgroup, row, rank): `choose` counts each workgroup's choices, `scan` turns
// them into each workgroup's first rank (one workgroup per expert), `place` hands out the slots.  Sums
// over rows are taken in a fixed order; the only atomics count in LDS, in whole numbers.
#include <algorithm>

#include "device.hpp"
#include "ft/train.hpp"

namespace ftrain::train {
namespace {

// Threads of a workgroup that chooses, of one of the backward pass.  Of 256 twice the workgroups choose, and
// their counts are twice as many: 131072 x 256, top 8 61.4 us, 59.9 with 512; 16384 x 64, top 2 10.5 and 10.2.
constexpr int kThreads = 512, kBackThreads = 256;
constexpr int kWaves   = kThreads / kWave;
constexpr int kCus     = 256;
// Most workgroups: as many as are on the chip at once with the registers of the widest rows.  Half as many
// again: choose 46.8, scan 9.7 and place 10.0 us at 131072 x 256 instead of 44.3, 7.6 and 7.7.
constexpr int kMaxBlocks = 2 * kCus;
// Which form the forward pass takes (moeRouteForward): passes of one workgroup over rows, and counts.
constexpr uint64_t kWholePasses = 2, kScanPasses = 4, kScanCounts = 32768;
// Workgroups of the form without `scan`.
constexpr int kMidBlocks = kCus;

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
    // Workspace: of each workgroup and expert, the choices (then their first rank) and the sum of p; of
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
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int j = 0; j < VPL; ++j) v[j] = -INFINITY;
    }
    // fetch: the loads alone, of what unpack makes logits of.
    static constexpr int kVec = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(kVec)));
    vec raw[VEC ? VPL / kVec : 1];
    T one[VEC ? 1 : VPL];
    __device__ __forceinline__ void fetch(const T* row, int n) {
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < VPL; j += kVec)
                if (index(j) < n) raw[j / kVec] = *reinterpret_cast<const vec*>(row + index(j));
        } else {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (index(j) < n) one[j] = row[index(j)];
        }
    }
    __device__ __forceinline__ void unpack(int n) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) v[j] = toFloat(VEC ? static_cast<T>(raw[VEC ? j / kVec : 0][j % kVec]) : one[VEC ? 0 : j]);
        if (n == G * VPL) return;
#pragma unroll
        for (int j = 0; j < VPL; ++j) v[j] = index(VEC ? j / kVec * kVec : j) < n ? v[j] : -INFINITY;
    }
    __device__ __forceinline__ void load(const T* row, int n) {
        fetch(row, n);
        unpack(n);
    }
    // Exponentials relative to `top` into p; their sum is returned: 0 only where every logit is minus
    // infinity (a NaN makes it NaN).
    __device__ __forceinline__ float exponentials(float (&p)[VPL], float top) const {
        const float base = top == -INFINITY ? 0.f : top;
        float total      = 0.f;
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            p[j] = expFast(v[j] - base);
            total += p[j];
        }
        return groupSum<G>(total);
    }
    __device__ __forceinline__ float largest() const {
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < VPL; ++j) m = fmaxf(m, v[j]);
        return groupMax<G>(m);
    }
};

__device__ __forceinline__ unsigned maxOf(unsigned a, unsigned b) { return a > b ? a : b; }

// The logits as whole numbers in their order, from which the largest are taken one by one (0: taken; a
// NaN counts as minus infinity, which is never chosen; the two zeros are one).  Integers, because a
// floating maximum of values that may be NaN takes two more instructions to make them quiet, at every
// step.  What a step costs is vector instructions of every lane for the one that holds the largest:
//   kPacked: a 16-bit logit leaves 13 bits of its number free, which hold 1023 less its index; the
// largest number is the largest logit with the lowest index, and each lane strikes it from its own.
//   kShared (16 logits a lane, or fp32 with lanes enough): the numbers lie in LDS in the row's order, a
// lane keeps the maximum of its run of them.  The lowest lane with the largest is found by a ballot, and
// the whole group reads that lane's run, one number each: a ballot finds the place, a maximum over the
// lanes is the run's next.
//   Otherwise (few lanes) the lowest index of those that are equal to the largest.
template <class T, int VPL, int G, bool VEC>
struct Candidates {
    static constexpr bool kPacked    = sizeof(T) == 2 && VPL == 8;
    static constexpr bool kShared    = !kPacked && G >= VPL;
    static constexpr unsigned kIndex = kMaxExperts - 1, kFree = 0x1FFFu;
    static constexpr unsigned kLeast = 0x00800000u;  // the number of the lowest finite value is not less
    // Words of a row in LDS: the rows of a wave start in different banks.  A lane's run lies in 16-byte
    // chunks, chunk c at place c ^ (lane / 4 mod 4) of every four, so that lanes write to different banks.
    static constexpr int kStride = G * VPL + 16;
    static __device__ __forceinline__ int placeOf(int run, int j) {
        constexpr int kMask = VPL / 4 - 1 < 3 ? VPL / 4 - 1 : 3;
        return run * VPL + (j ^ (run & 4 * kMask));
    }
    unsigned key[VPL];
    unsigned own;          // the lane's largest
    unsigned* const row_;  // kShared: the row's numbers

    __device__ __forceinline__ Candidates(const Row<T, VPL, G, VEC>& row, unsigned* lds) : row_(lds + threadIdx.x / G * kStride) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) {
            const unsigned bits = __builtin_bit_cast(unsigned, fmaxf(row.v[j] + 0.f, -INFINITY));
            unsigned k          = bits ^ (static_cast<unsigned>(static_cast<int>(bits) >> 31) | 0x80000000u);
            if constexpr (kPacked) k = (k & ~kFree) | (kIndex - row.index(j));
            key[j] = k;
        }
        if constexpr (kShared) {
            waveFence();  // the wave is done with the rows before
            typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
            if constexpr (VEC) {
#pragma unroll
                for (int j = 0; j < VPL; j += 4)
                    *reinterpret_cast<u32x4*>(row_ + placeOf(row.g, j)) = u32x4{key[j], key[j + 1], key[j + 2], key[j + 3]};
            } else {
#pragma unroll
                for (int j = 0; j < VPL; ++j) row_[placeOf(row.index(j) / VPL, row.index(j) % VPL)] = key[j];
                waveFence();
#pragma unroll
                for (int j = 0; j < VPL; j += 4) {
                    const u32x4 x = *reinterpret_cast<const u32x4*>(row_ + placeOf(row.g, j));
#pragma unroll
                    for (int e = 0; e < 4; ++e) key[j + e] = x[e];
                }
            }
            waveFence();
        }
        own = mine();
    }
    __device__ __forceinline__ unsigned mine() const {
        unsigned m = key[0];
#pragma unroll
        for (int j = 1; j < VPL; ++j) m = maxOf(m, key[j]);
        return m;
    }
    // The group's largest number.
    __device__ __forceinline__ unsigned best() const { return largest(own); }
    static __device__ __forceinline__ unsigned largest(unsigned v) {
        return groupReduce<G>(v, [](unsigned a, unsigned b) { return maxOf(a, b); });
    }
    static __device__ __forceinline__ float value(unsigned k) {
        if (k < kLeast) return -INFINITY;
        if constexpr (kPacked) k = (k & 0x80000000u) ? k & ~kFree : k | kFree;
        return __builtin_bit_cast(float, (k & 0x80000000u) ? k ^ 0x80000000u : ~k);
    }
    // The lowest lane of the group for which `is` holds (for one it does).
    static __device__ __forceinline__ int lowestLane(bool is, int g) {
        const unsigned long long all = __ballot(is);
        if constexpr (G == kWave) return __builtin_ctzll(all);
        const int first = threadIdx.x % kWave - g;
        if constexpr (G == 32) return __builtin_ctz(static_cast<unsigned>(first == 0 ? all : all >> 32));
        return __builtin_ctz(static_cast<unsigned>(all >> first));
    }
    // Takes out the largest, `best`; returns its index.
    __device__ __forceinline__ int take(unsigned best, const Row<T, VPL, G, VEC>& row) {
        if constexpr (kPacked) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) key[j] = key[j] == best ? 0u : key[j];
            own = mine();
            return kIndex - (best & kIndex);
        } else if constexpr (kShared) {
            const int from = lowestLane(own == best, row.g);
            unsigned* const mine = row_ + placeOf(from, row.g % VPL);
            unsigned x           = row.g < VPL ? *mine : 0u;
            const int j          = lowestLane(x == best && row.g < VPL, row.g);
            x                    = row.g == j ? 0u : x;
            if (row.g == j) *mine = 0u;
            waveFence();
            const unsigned next = largest(x);
            own                 = row.g == from ? next : own;
            return from * VPL + j;
        } else {
            int found = INT32_MAX;
#pragma unroll
            for (int j = VPL - 1; j >= 0; --j)
                if (key[j] == best) found = row.index(j);
            const int at = groupReduce<G>(found, [](int a, int b) { return min(a, b); });
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (row.index(j) == at) key[j] = 0u;
            own = mine();
            return at;
        }
    }
};

// Of a workgroup's threads, what each adds to the routed rows, the choices and sum_e counts_e sum_t p_te:
// the launch's results from them.
template <int THREADS>
__device__ __forceinline__ void finishLoss(const RouteArgs& a, int routed, int choices, float dot) {
    constexpr int kWaves = THREADS / kWave;
    __shared__ int of_routed[kWaves], of_choices[kWaves];
    __shared__ float of_dot[kWaves];
    routed         = groupSum<kWave>(routed);
    choices        = groupSum<kWave>(choices);
    dot            = groupSum<kWave>(dot);
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) of_routed[wave] = routed, of_choices[wave] = choices, of_dot[wave] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) routed += of_routed[w], choices += of_choices[w], dot += of_dot[w];
        *a.routed = routed;
        *a.loss   = static_cast<float>(a.n_experts) * (dot / static_cast<float>(max(choices, 1))) / static_cast<float>(max(routed, 1));
    }
}

// What `choose` and `place` keep in LDS (one workgroup may do both, one after the other).
struct ChooseLds {
    alignas(16) unsigned rows[kThreads * 16 + kThreads];  // Candidates: at most 64 rows, 16 words apart
};
template <int THREADS>
struct PlaceLds {
    int first[kMaxExperts];                  // slot of the workgroup's first choice of each expert
    int next[THREADS / kWave][kMaxExperts];  // each wave's choices, then its next slot
};

// hist: the workgroup's choices of each expert.  choices: where one workgroup has all rows, what it chose,
// for it to place from LDS (64 x 8: 8.5 us with counts and choices through memory, 5.1 so).
template <class T, int VPL, int G, bool VEC>
__device__ __forceinline__ void chooseRows(const RouteArgs& a, ChooseLds& lds, int* hist, int16_t* choices) {
    constexpr int kRows = kThreads / G;  // rows at a time
    const bool whole    = a.blocks == 1;
    const int group = threadIdx.x / G, n = a.n_experts;
    Row<T, VPL, G, VEC> row;
    row.g = threadIdx.x % G;
    for (int e = threadIdx.x; e < n; e += kThreads) hist[e] = 0;
    __syncthreads();

    float sum_p[VPL] = {};
    int routed       = 0;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.rows_per_block;
    const int64_t last  = min(first + a.rows_per_block, a.rows);
    // The next row's loads are under way while a row is worked on.
    bool kept        = false;
    const auto fetch = [&](int64_t t) {
        if (t >= last) return;
        kept = a.mask == nullptr || a.mask[t] != 0;
        row.fetch(static_cast<const T*>(a.logits) + t * a.ld, n);
    };
    fetch(first + group);
    for (int64_t t = first + group; t < last; t += kRows) {
        int32_t* const experts = a.experts + t * a.top_k;
        float* const gates     = a.gates + t * a.top_k;
        if (kept)
            row.unpack(n);
        else
            row.clear();
        fetch(t + kRows);
        Candidates<T, VPL, G, VEC> left(row, lds.rows);
        unsigned best   = left.best();
        const float top = left.value(best);
        float p[VPL];
        const float total = row.exponentials(p, top);
        if (total == 0.f) {
            for (int k = row.g; k < a.top_k; k += G) {
                experts[k] = -1;
                gates[k]   = 0.f;
                if (whole) choices[t * a.top_k + k] = -1;
            }
            continue;
        }
        const float inv = 1.f / total;
#pragma unroll
        for (int j = 0; j < VPL; ++j) sum_p[j] += p[j] * inv;
        ++routed;
        // Lane g keeps choices g, g + G ..
        constexpr int kSlots = VPL < kMaxTopK / G ? VPL : G < kMaxTopK ? kMaxTopK / G : 1;
        float gate[kSlots], chosen = 0.f;
        int at[kSlots];
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
            at[s]   = INT32_MAX;
            gate[s] = 0.f;
            if (s * G >= a.top_k) continue;
            unsigned number = 0;
            for (int k = 0; k < G && s * G + k < a.top_k; ++k) {
                const int e = left.take(best, row);
                if (k == row.g) at[s] = best >= left.kLeast ? e : INT32_MAX, number = best;
                best = left.best();
            }
            // A row whose sum is NaN has NaN gates.
            gate[s] = at[s] < n ? expExact(left.value(number) - top) * inv : 0.f;
            chosen += gate[s];
        }
        if (a.normalize) {
            const float scale = 1.f / groupSum<G>(chosen);
#pragma unroll
            for (int s = 0; s < kSlots; ++s) gate[s] = at[s] < n ? gate[s] * scale : 0.f;
        }
#pragma unroll
        for (int s = 0; s < kSlots; ++s) {
            const int k = s * G + row.g;
            if (k < a.top_k) {
                const int e = at[s] < n ? at[s] : -1;
                experts[k]  = e;
                gates[k]    = gate[s];
                if (e >= 0) atomicAdd(&hist[e], 1);
                if (whole) choices[t * a.top_k + k] = static_cast<int16_t>(e);
            }
        }
    }
    // Each wave's rows, then the waves.
#pragma unroll
    for (int j = 0; j < VPL; ++j) sum_p[j] = acrossGroups<G>(sum_p[j]);
    routed = row.g == 0 ? routed : 0;
    __syncthreads();
    float* const sums = reinterpret_cast<float*>(lds.rows);  // [kWaves][G * VPL]
    if (threadIdx.x % kWave < G) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) sums[threadIdx.x / kWave * (G * VPL) + row.index(j)] = sum_p[j];
    }
    __syncthreads();
    int chosen = 0;
    float dot  = 0.f;
    for (int e = threadIdx.x; e < n; e += kThreads) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += sums[w * (G * VPL) + e];
        const int c = hist[e];
        if (whole) {
            a.counts[e] = c;
            chosen += c;
            dot += static_cast<float>(c) * sum;
        } else {
            a.block_count[static_cast<int64_t>(blockIdx.x) * n + e] = c;
            a.block_p[static_cast<int64_t>(blockIdx.x) * n + e]     = sum;
        }
    }
    if (whole) {
        finishLoss<kThreads>(a, routed, chosen, dot);
    } else {
        __shared__ int of_waves[kWaves];
        routed = groupSum<kWave>(routed);
        if (threadIdx.x % kWave == 0) of_waves[threadIdx.x / kWave] = routed;
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
            for (int w = 1; w < kWaves; ++w) routed += of_waves[w];
            a.block_routed[blockIdx.x] = routed;
        }
    }
}

// Exclusive prefix sum of one value a thread over the workgroup; total: the sum.
template <int THREADS>
__device__ __forceinline__ int blockScan(int v, int& total) {
    constexpr int kWaves = THREADS / kWave;
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

// Of kScanExperts experts: each workgroup's first rank in place of its count, the expert's count, its sum
// of p.  Adjacent threads take adjacent experts, each a run of the workgroups; runs are joined in groups.
constexpr int kScanExperts = 8, kScanThreads = 1024, kScanGroup = 8;
__global__ __launch_bounds__(kScanThreads) void scan(RouteArgs a) {
    constexpr int kRuns = kScanThreads / kScanExperts, kGroups = kRuns / kScanGroup;
    constexpr int kPer = kMaxBlocks / kRuns;
    __shared__ int counts[kRuns][kScanExperts], groups[kGroups][kScanExperts];
    __shared__ float sums[kRuns][kScanExperts], group_sums[kGroups][kScanExperts];
    const int n = a.n_experts, run = threadIdx.x / kScanExperts, i = threadIdx.x % kScanExperts;
    const int e = blockIdx.x * kScanExperts + i, first = run * kPer;
    int32_t* const count = a.block_count + e;
    const float* const p = a.block_p + e;
    int mine[kPer], c = 0;
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < kPer; ++b) {
        const bool in = e < n && first + b < a.blocks;
        mine[b]       = in ? count[static_cast<int64_t>(first + b) * n] : 0;
        sum += in ? p[static_cast<int64_t>(first + b) * n] : 0.f;
    }
#pragma unroll
    for (int b = 0; b < kPer; ++b) c += mine[b];
    counts[run][i] = c;
    sums[run][i]   = sum;
    __syncthreads();
    if (run < kGroups) {
        int all   = 0;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < kScanGroup; ++r) {
            all += counts[run * kScanGroup + r][i];
            sum += sums[run * kScanGroup + r][i];
        }
        groups[run][i]     = all;
        group_sums[run][i] = sum;
    }
    __syncthreads();
    const int group = run / kScanGroup;
    int before      = 0;
    for (int q = 0; q < group; ++q) before += groups[q][i];
    for (int r = group * kScanGroup; r < run; ++r) before += counts[r][i];
    if (run == kRuns - 1 && e < n) {
        float all = 0.f;
        for (int q = 0; q < kGroups; ++q) all += group_sums[q][i];
        a.counts[e] = before + c;
        a.sum_p[e]  = all;
    }
#pragma unroll
    for (int b = 0; b < kPer; ++b) {
        if (e < n && first + b < a.blocks) count[static_cast<int64_t>(first + b) * n] = before;
        before += mine[b];
    }
}

// Where the counts are from which the slots follow: the only workgroup's own; those of each workgroup, which
// every one adds up by itself; what `scan` has made of these.
enum class Counts { kOwn, kEach, kScanned };
// kEach: of how many threads an expert's counts are added up.
template <int THREADS>
__device__ __forceinline__ int partsOf(int experts) {
    return experts <= THREADS / 8 ? 8 : experts <= THREADS / 2 ? 2 : 1;
}

// The slots of the workgroup's choices.  kOwn: with the choices and their counts from LDS.
template <Counts FORM, int THREADS>
__device__ __forceinline__ void placeRows(const RouteArgs& a, PlaceLds<THREADS>& lds, const int* own, const int16_t* choices) {
    constexpr int kThreads = THREADS, kWaves = THREADS / kWave;
    int* const first = lds.first;
    auto& next       = lds.next;
    const int n = a.n_experts, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.rows_per_block * a.top_k;
    const int64_t end   = min(begin + static_cast<int64_t>(a.rows_per_block) * a.top_k, a.rows * a.top_k);
    const int per_wave  = static_cast<int>((end - begin + kThreads - 1) / kThreads) * kWave;
    const int64_t mine = min(begin + static_cast<int64_t>(wave) * per_wave, end), stop = min(mine + per_wave, end);
    auto chosen = [&](int64_t i) -> int { return i >= stop ? -1 : FORM == Counts::kOwn ? choices[i] : a.experts[i]; };
    const int ahead = chosen(mine + lane);  // under way with the counts
    if constexpr (FORM == Counts::kEach) {
        // A thread an expert, or several: adjacent threads adjacent experts, each with the workgroups
        // from `part` on in steps of `parts`.
        const int parts = partsOf<kThreads>(n), part = threadIdx.x / (kThreads / parts), self = blockIdx.x;
        __shared__ int all_of[kThreads], before_of[kThreads];
        for (int e0 = 0; e0 < n; e0 += kThreads / parts) {
            const int e = e0 + threadIdx.x % (kThreads / parts);
            int all = 0, before = 0;
            if (e < n) {
#pragma unroll 16
                for (int b = part; b < a.blocks; b += parts) {
                    const int c = a.block_count[static_cast<int64_t>(b) * n + e];
                    all += c;
                    before += b < self ? c : 0;
                }
            }
            all_of[threadIdx.x]    = all;
            before_of[threadIdx.x] = before;
            __syncthreads();
            if (part == 0 && e < n) {
                for (int q = 1; q < parts; ++q) {
                    all += all_of[threadIdx.x + q * (kThreads / parts)];
                    before += before_of[threadIdx.x + q * (kThreads / parts)];
                }
                next[0][e] = all;
                next[1][e] = before;
            }
            __syncthreads();
        }
    }
    auto count_of = [&](int e) { return FORM == Counts::kOwn ? own[e] : FORM == Counts::kEach ? next[0][e] : a.counts[e]; };
    auto before_of = [&](int e) {
        return FORM == Counts::kOwn    ? 0
               : FORM == Counts::kEach ? next[1][e]
                                       : a.block_count[static_cast<int64_t>(blockIdx.x) * n + e];
    };
    int before = 0;
    for (int e0 = 0; e0 < n; e0 += kThreads) {
        const int e = e0 + threadIdx.x;
        int total;
        const int of_blocks = e < n ? before_of(e) : 0;
        const int at        = blockScan<THREADS>(e < n ? count_of(e) : 0, total);
        if (e < n) first[e] = before + at + of_blocks;
        before += total;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n; e += kThreads)
        for (int w = 0; w < kWaves; ++w) next[w][e] = 0;
    __syncthreads();
    for (int64_t i0 = mine; i0 < stop; i0 += kWave) {
        const int e = i0 == mine ? ahead : chosen(i0 + lane);
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
        const int e     = i0 == mine ? ahead : chosen(i);
        // The lanes with the same expert: agreement in every bit of its index.
        unsigned long long peers = __ballot(e >= 0);
        for (int bit = 1; bit < n; bit <<= 1) {
            const unsigned long long set = __ballot((e & bit) != 0);
            peers &= (e & bit) ? set : ~set;
        }
        int slot = -1;
        if (e >= 0) slot = next[wave][e] + __popcll(peers & ((1ull << lane) - 1ull));
        // Every lane has read before the last of each expert's lanes writes, and the next round reads
        // after it.
        waveFence();
        if (e >= 0 && (peers >> lane) == 1ull) next[wave][e] = slot + 1;
        waveFence();
        if (i < stop) a.slots[i] = slot;
    }
}

// The routed rows and the loss, by a workgroup of its own; without `scan` also the counts.
template <bool SCANNED, int THREADS>
__device__ __forceinline__ void lossOfBlocks(const RouteArgs& a) {
    const int n = a.n_experts;
    int routed = 0, choices = 0;
    float dot = 0.f;
    for (int b = threadIdx.x; b < a.blocks; b += THREADS) routed += a.block_routed[b];
    if constexpr (SCANNED) {
        for (int e = threadIdx.x; e < n; e += THREADS) {
            const int c = a.counts[e];
            choices += c;
            dot += static_cast<float>(c) * a.sum_p[e];
        }
    } else {
        const int parts = partsOf<THREADS>(n), part = threadIdx.x / (THREADS / parts);
        __shared__ int all_of[THREADS];
        __shared__ float sum_of[THREADS];
        for (int e0 = 0; e0 < n; e0 += THREADS / parts) {
            const int e = e0 + threadIdx.x % (THREADS / parts);
            int all     = 0;
            float sum   = 0.f;
            if (e < n) {
#pragma unroll 16
                for (int b = part; b < a.blocks; b += parts) {
                    all += a.block_count[static_cast<int64_t>(b) * n + e];
                    sum += a.block_p[static_cast<int64_t>(b) * n + e];
                }
            }
            all_of[threadIdx.x] = all;
            sum_of[threadIdx.x] = sum;
            __syncthreads();
            if (part == 0 && e < n) {
                for (int q = 1; q < parts; ++q) {
                    all += all_of[threadIdx.x + q * (THREADS / parts)];
                    sum += sum_of[threadIdx.x + q * (THREADS / parts)];
                }
                a.counts[e] = all;
                choices += all;
                dot += static_cast<float>(all) * sum;
            }
            __syncthreads();
        }
    }
    finishLoss<THREADS>(a, routed, choices, dot);
}

// One workgroup that has all rows goes on to place them.
template <class T, int VPL, int G, bool VEC>
__global__ __launch_bounds__(kThreads) void choose(RouteArgs a) {
    __shared__ int hist[kMaxExperts];
    __shared__ union {
        ChooseLds choose;
        PlaceLds<kThreads> place;
    } lds;
    extern __shared__ int16_t choices[];  // one workgroup: rows x top_k
    chooseRows<T, VPL, G, VEC>(a, lds.choose, hist, choices);
    if (a.blocks > 1) return;
    __syncthreads();
    placeRows<Counts::kOwn, kThreads>(a, lds.place, hist, choices);
}

// 131072 x 256, top 8 (16384 x 64, top 2): 8.3 us (8.1) with 256 threads, 7.4 (6.9) with 512, 10.8 (10.7)
// with 1024; 7.1 (5.4) with 512, the choices under way with the counts and the loss to a workgroup of its own.
constexpr int kPlaceThreads = 512;
template <bool SCANNED>
__global__ __launch_bounds__(kPlaceThreads) void place(RouteArgs a) {
    if (static_cast<int>(blockIdx.x) == a.blocks) {
        lossOfBlocks<SCANNED, kPlaceThreads>(a);
        return;
    }
    __shared__ PlaceLds<kPlaceThreads> lds;
    placeRows<SCANNED ? Counts::kScanned : Counts::kEach, kPlaceThreads>(a, lds, nullptr, nullptr);
}

template <class T, int VPL, int G, bool VEC>
__global__ __launch_bounds__(kBackThreads) void backward(RouteArgs a) {
    constexpr int kRows = kBackThreads / G;
    // Of each group's row: p, and what its choices add to the gradient.
    __shared__ __attribute__((aligned(16))) float row_p[kBackThreads * VPL], row_add[kBackThreads * VPL];
    const int group = threadIdx.x / G, n = a.n_experts;
    Row<T, VPL, G, VEC> row;
    row.g              = threadIdx.x % G;
    float* const all_p = row_p + group * (G * VPL);
    float* const add   = row_add + group * (G * VPL);
    int total = 0, all;
    for (int e = threadIdx.x; e < n; e += kBackThreads) total += a.counts[e];
    (void)blockScan<kBackThreads>(total, all);
    // d loss / d p_te
    const float factor = *a.grad_loss * static_cast<float>(n) / static_cast<float>(max(all, 1)) /
                         static_cast<float>(max(*a.routed, 1));
    float balance[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j)
        balance[j] = row.index(j) < n ? factor * static_cast<float>(a.counts[row.index(j)]) : 0.f;

    const int64_t stride = static_cast<int64_t>(gridDim.x) * kRows, first = static_cast<int64_t>(blockIdx.x) * kRows + group;
    // The next row's loads are under way while a row is worked on: its logits and the lane's first choice
    // (100003 x 160 fp32, six choices: 33.3 -> 31.9 us).
    bool kept        = false;
    int next_expert  = -1;
    float next_grad  = 0.f;
    const auto fetch = [&](int64_t t) {
        if (t >= a.rows) return;
        kept = a.mask == nullptr || a.mask[t] != 0;
        row.fetch(static_cast<const T*>(a.logits) + t * a.ld, n);
        if (row.g < a.top_k) {
            next_expert = a.experts[t * a.top_k + row.g];
            next_grad   = a.grad_gates[t * a.top_k + row.g];
        }
    };
    fetch(first);
    for (int64_t t = first; t < a.rows; t += stride) {
        T* const out = static_cast<T*>(a.grad_logits) + t * a.grad_ld;
        float p[VPL], d[VPL] = {}, sum = 0.f;
        const bool routed      = kept;
        const int first_expert = next_expert;
        const float first_grad = next_grad;
        row.unpack(n);
        fetch(t + stride);
        if (routed) sum = row.exponentials(p, row.largest());
        if (sum != 0.f) {
            const int32_t* const experts = a.experts + t * a.top_k;
            const float* const grads     = a.grad_gates + t * a.top_k;
            const float inv              = 1.f / sum;
            // f(expert, gradient of its gate) of the lane's choices.
            const auto eachChoice = [&](auto&& f) {
                for (int k = row.g; k < a.top_k; k += G) {
                    const int e = k < G ? first_expert : experts[k];
                    if (e >= 0 && e < n) f(e, k < G ? first_grad : grads[k]);
                }
            };
            // The choices reach their experts' lanes through LDS (a comparison of every choice with
            // every logit took most of the kernel: 100003 x 160, six choices, 46 -> 33 us).
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                p[j] *= inv;
                add[row.index(j)] = 0.f;
                if (a.normalize) all_p[row.index(j)] = p[j];
            }
            waveFence();
            float picked = 0.f, weighted = 0.f;
            if (a.normalize) {
                // Of the chosen: sum of p, and sum of p dgate.
                eachChoice([&](int e, float g) {
                    picked += all_p[e];
                    weighted += all_p[e] * g;
                });
                picked   = groupSum<G>(picked);
                weighted = groupSum<G>(weighted);
            }
            eachChoice([&](int e, float g) { add[e] = a.normalize ? all_p[e] / picked * (g - weighted / picked) : g; });
            waveFence();
            float dot = 0.f, more[VPL];
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                more[j] = add[row.index(j)];
                d[j]    = a.normalize ? balance[j] : balance[j] + more[j];
                dot += p[j] * d[j];
            }
            waveFence();
            dot = groupSum<G>(dot);
#pragma unroll
            for (int j = 0; j < VPL; ++j) d[j] = p[j] * (d[j] - dot) + (a.normalize ? more[j] : 0.f);
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
    const integral_constant<int, 16> sixteen;
    if (n <= 8) return pick(integral_constant<int, 1>{}, eight);
    if (n <= 16) return pick(integral_constant<int, 2>{}, eight);
    if (n <= 32) return pick(integral_constant<int, 4>{}, eight);
    if (n <= 64) return pick(integral_constant<int, 8>{}, eight);
    if (n <= 128) return pick(integral_constant<int, 16>{}, eight);
    // Backward has no steps across lanes to share, and is bound by memory with eight a lane (100003 x 160
    // fp32: 33 us, with 16 a lane 45).
    if constexpr (BACK) {
        if (n <= 256) return pick(integral_constant<int, 32>{}, eight);
        if (n <= 512) return pick(integral_constant<int, 64>{}, eight);
    } else {
        if (n <= 256) return pick(integral_constant<int, 16>{}, sixteen);
        if (n <= 512) return pick(integral_constant<int, 32>{}, sixteen);
    }
    return pick(integral_constant<int, 64>{}, sixteen);
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
    // Whole passes of the workgroup over its rows, in one of three forms:
    //   few passes in all: one workgroup does everything, in one launch.  us of the device in one launch
    //     of one pass and of two, against two launches: 8 experts, top 2 6.4, 8.7 / 8.4; 64, top 2 5.6,
    //     6.8 / 7.4; 64 fp32, top 8 6.8, 9.4 / 8.9; 256, top 8 7.8, 10.5 / 12.3; 1024, top 8 8.9, 12.2 /
    //     13.7 (and the host's 2.4 for a launch);
    //   as many workgroups as CUs, while the counts that each of `place` then reads (one of every
    //     workgroup and expert) stay few: two launches (16384 x 64: 15.2 us in three, 13.5 in two);
    //   two workgroups on each CU, and `scan` between.
    const uint64_t at_once = kThreads / lanes, all = ceilDiv(a.rows, at_once);
    const bool whole       = all <= kWholePasses;
    const bool scanned     = !whole && (all > kScanPasses * kMidBlocks || p.logits.cols * kMidBlocks > kScanCounts);
    const uint64_t passes  = whole ? std::max<uint64_t>(1, all) : ceilDiv(all, scanned ? kMaxBlocks : kMidBlocks);
    a.rows_per_block       = static_cast<int32_t>(passes * at_once);
    a.blocks               = static_cast<int32_t>(std::max<uint64_t>(1, ceilDiv(a.rows, a.rows_per_block)));
    a.block_count          = static_cast<int32_t*>(workspace);
    a.block_p              = reinterpret_cast<float*>(a.block_count + p.logits.cols * kMaxBlocks);
    a.block_routed         = reinterpret_cast<int32_t*>(a.block_p + p.logits.cols * kMaxBlocks);
    a.sum_p                = reinterpret_cast<float*>(a.block_routed + kMaxBlocks);
    launchWithLds(kernel, "router choose", dim3(a.blocks), dim3(kThreads), whole ? a.rows * a.top_k * sizeof(int16_t) : 0, stream, a);
    if (a.blocks == 1) return;
    if (scanned) {
        launch(&scan, "router scan", dim3(static_cast<uint32_t>(ceilDiv(a.n_experts, kScanExperts))), dim3(kScanThreads), stream, a);
        launch(&place<true>, "router place", dim3(a.blocks + 1), dim3(kPlaceThreads), stream, a);
    } else {
        launch(&place<false>, "router place", dim3(a.blocks + 1), dim3(kPlaceThreads), stream, a);
    }
}

void moeRouteBackward(const MoeRoute& p, hipStream_t stream) {
    RouteArgs a = arguments(p);
    if (a.rows == 0) return;
    int lanes = 0;
    const bool vec = vectorRows(p.logits, p.type) && vectorRows(p.grad_logits, p.type);
    const Kernel kernel    = kernelFor<true>(p.type, vec, static_cast<int>(p.logits.cols), lanes);
    const uint64_t at_once = kBackThreads / lanes;
    launch(kernel, "router backward", dim3(static_cast<uint32_t>(std::min<uint64_t>(ceilDiv(a.rows, at_once), 8 * kCus))),
           dim3(kBackThreads), stream, a);
}

}  // namespace ftrain::train
