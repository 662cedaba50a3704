// The output head's product with softmax cross entropy, and its gradients.  With x the hidden states
// (tokens x hidden), w the weight (classes x hidden), y the targets, g the losses' gradients:
//   l = x w^T, lse_t = log sum_v exp l_tv, loss_t = lse_t - l_t,y(t);
//   dl_tv = g_t (exp(l_tv - lse_t) - [v = y_t]), dx = dl w, dw = dl^T x.
// l and dl (tokens x classes) are never kept whole: forward, a tile of l is reduced where it was
// computed to each row's maximum and sum of exponentials over the tile's classes; backward, l is
// formed again in pieces of the classes, a piece of dl goes to the workspace and is used for both
// products.
//
// A token whose target is the ignored index takes no part: the others' rows of x are packed densely
// first, so neither its hidden state (whatever is in it) nor its work reaches any sum.  Where x lies
// and how it is aligned is thereby settled too.  (The loss of few tokens goes without: Layout::direct.)
// A target outside the classes makes its token's loss and gradients NaN.
#include <algorithm>

#include "cross_entropy.hpp"
#include "device.hpp"
#include "ft/train.hpp"

namespace ftrain::train {
namespace {

constexpr int kThreads     = 256;
constexpr int kPackThreads = 512;
constexpr int kFinishThreads = 1024;
// Most workgroups that pack: two on each of the 256 CUs.
constexpr int kPackBlocks = 512;

struct PackArgs {
    Targets targets;
    int64_t tokens;
    const float *lse, *grad_loss;  // backward
    Head* head;
    int32_t* place;  // each token's packed row, -1 if ignored
    RowInfo* rows;
    const void* x;
    void* packed;
    int64_t ld, cols, padded;
    int64_t per_block;  // tokens
    int pair;           // packed rows of each (kFewTokens)
    bool backward, scaled;
};

// A row of `cols` elements at any address, padded with zeros, by one wave; out: whole 16-byte units.
template <class T>
__device__ __forceinline__ void copyRow(const T* from, T* out, int64_t cols, int64_t padded) {
    constexpr int N     = Pack<T>::kCount;
    const int lane      = threadIdx.x % kWave;
    const int64_t whole = cols / N * N;
#pragma unroll 4
    for (int64_t i = lane * N; i < whole; i += kWave * N)
        *reinterpret_cast<Pack<T>*>(out + i) = *reinterpret_cast<const Pack<T>*>(from + i);
    if (whole + lane < padded) out[whole + lane] = whole + lane < cols ? from[whole + lane] : static_cast<T>(0.f);
}

// The kept tokens' rows of x, in order and densely.  A workgroup takes `per_block` tokens; it counts the
// kept ones before them by itself, so that one launch does what a scan and a copy would: 8192 x 4096 bf16
// 38 us in two launches, 28 in one (134 MB at 4.8 TB/s).
template <class T>
__global__ __launch_bounds__(kPackThreads) void packTokens(PackArgs a) {
    constexpr int kWaves = kPackThreads / kWave;
    __shared__ int wave_count[kWaves];
    __shared__ float wave_max[kWaves];
    __shared__ int place[kPackThreads];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    auto kept = [&](int64_t t, int64_t& y) {
        y = a.targets.given(t);
        return y != a.targets.ignore_index;
    };
    const int64_t first = blockIdx.x * a.per_block, last = min(first + a.per_block, a.tokens);
    int64_t y;
    int count = 0;
    float top = 0.f;
#pragma unroll 4
    for (int64_t t = threadIdx.x; t < first; t += kPackThreads) count += kept(t, y);
    if (a.scaled)
        for (int64_t t = threadIdx.x; t < a.tokens; t += kPackThreads)
            if (kept(t, y)) top = fmaxf(top, fabsf(a.grad_loss[t]));
    count = groupSum<kWave>(count);
    top   = groupMax<kWave>(top);
    if (lane == 0) {
        wave_count[wave] = count;
        wave_max[wave]   = top;
    }
    __syncthreads();
    int before = 0;
    for (int w = 0; w < kWaves; ++w) {
        before += wave_count[w];
        top = fmaxf(top, wave_max[w]);
    }
    // fp16 holds no small probability: dl is kept times the power of two that brings the largest |g| into
    // [2^14, 2^15); |dl| <= |g| stays below fp16's largest value, and what is lost is below 2^-39 of the
    // largest g.
    float scale = 1.f;
    if (a.scaled && top > 0.f && top < INFINITY) {
        int e;
        (void)frexpf(top, &e);  // top in [2^(e-1), 2^e)
        scale = ldexpf(1.f, min(15 - e, 120));
    }
    for (int64_t t0 = first; t0 < last; t0 += kPackThreads) {
        const int64_t t  = t0 + threadIdx.x;
        const bool keeps = t < last && kept(t, y);
        const unsigned long long mask = __ballot(keeps);
        __syncthreads();
        if (lane == 0) wave_count[wave] = __popcll(mask);
        __syncthreads();
        int at = before + __popcll(mask & ((1ull << lane) - 1ull));
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) at += wave_count[w];
            before += wave_count[w];
        }
        place[threadIdx.x] = keeps ? at : -1;
        if (t < last) {
            a.place[t] = keeps ? at : -1;
            if (keeps)
                a.rows[at] = RowInfo{a.backward ? a.lse[t] : 0.f, a.backward ? a.grad_loss[t] * scale : 0.f,
                                     y >= 0 && y < a.targets.classes ? static_cast<int32_t>(y) : -1};
        }
        __syncthreads();
        for (int64_t i = wave; i < min(last - t0, static_cast<int64_t>(kPackThreads)); i += kWaves)
            if (place[i] >= 0)
                for (int q = 0; q < a.pair; ++q)
                    copyRow(static_cast<const T*>(a.x) + (t0 + i) * a.ld,
                            static_cast<T*>(a.packed) + (static_cast<int64_t>(place[i]) * a.pair + q) * a.padded, a.cols, a.padded);
    }
    if (threadIdx.x == 0 && blockIdx.x == gridDim.x - 1) *a.head = Head{before, scale, 1.f / scale};
}

// A piece of the weight in rows of whole 16-byte units.
template <class T>
__global__ __launch_bounds__(kThreads) void packWeight(const T* w, int64_t ld, int64_t rows, int64_t cols, T* out, int64_t padded) {
    constexpr int kWaves = kThreads / kWave;
    for (int64_t v = static_cast<int64_t>(blockIdx.x) * kWaves + threadIdx.x / kWave; v < rows; v += static_cast<int64_t>(gridDim.x) * kWaves)
        copyRow(w + v * ld, out + v * padded, cols, padded);
}

// Four adjacent sums over the slices first, first + step .. below `end`; at(z): where slice z's are.  Four
// loads are under way at once, the first again for those past the end (one after the other, the six slices
// of 500 x 1024 took 5.6 us, so 4.9).
template <class AT>
__device__ __forceinline__ float4 sumSlices(int first, int step, int end, AT&& at) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (first < end && first + step >= end) return *reinterpret_cast<const float4*>(at(first));
    for (int z0 = first; z0 < end; z0 += 4 * step) {
        float4 x[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) x[b] = *reinterpret_cast<const float4*>(at(z0 + b * step < end ? z0 + b * step : z0));
#pragma unroll
        for (int b = 0; b < 4; ++b)
            if (z0 + b * step < end) s.x += x[b].x, s.y += x[b].y, s.z += x[b].z, s.w += x[b].w;
    }
    return s;
}

// Four adjacent logits, of which `left` lie in the matrix (none: nothing is read).
__device__ __forceinline__ void joinSlices(const float* from, int64_t slice, int slices, int left, float (&v)[4]) {
    const float4 s = left > 0 ? sumSlices(0, 1, slices, [&](int z) { return from + z * slice; }) : make_float4(0.f, 0.f, 0.f, 0.f);
    v[0] = s.x, v[1] = s.y, v[2] = s.z, v[3] = s.w;
}

// Where k is cut (Tiling), the logits' slices joined, four adjacent classes a lane and a wave 256 of a
// row: its maximum and sum of exponentials over them, and the target's logit.
__global__ __launch_bounds__(kThreads) void joinLogSum(const float* logits, int64_t ld, int64_t slice, int slices,
                                                       const Head* head, Targets targets, int n, int first_class,
                                                       int64_t tokens, float2* part, float* hit) {
    const int64_t row = static_cast<int64_t>(blockIdx.y) * (kThreads / kWave) + threadIdx.x / kWave;
    const int col     = blockIdx.x * 256 + 4 * (threadIdx.x % kWave);
    if (row >= (head == nullptr ? tokens : head->valid)) return;
    float v[4];
    joinSlices(logits + row * ld + col, slice, slices, n - col, v);
    const int at = targets(row) - first_class - col;
    float top    = -INFINITY;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (col + e >= n) v[e] = -INFINITY;
        if (e == at && col + e < n) hit[row] = v[e];
        top = fmaxf(top, v[e]);
    }
    top              = groupMax<kWave>(top);
    const float base = top == -INFINITY ? 0.f : top;
    float sum        = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += expFast(v[e] - base);
    sum = groupSum<kWave>(sum);
    if (threadIdx.x % kWave == 0) part[(first_class / 256 + blockIdx.x) * tokens + row] = make_float2(top, sum);
}

// The same for dl, with zeros up to `padded` columns.
template <class T>
__global__ __launch_bounds__(kThreads) void joinGradLogits(const float* logits, int64_t ld, int64_t slice, int slices,
                                                           const Head* head, const RowInfo* rows, int n, int padded,
                                                           int first_class, T* dl, int64_t ldd, int pair) {
    const int64_t row = static_cast<int64_t>(blockIdx.y) * (kThreads / kWave) + threadIdx.x / kWave;
    const int col     = blockIdx.x * 256 + 4 * (threadIdx.x % kWave);
    if (row >= head->valid || col >= padded) return;
    float v[4];
    joinSlices(logits + row * ld + col, slice, slices, n - col, v);
    const RowInfo r = rows[row];
    const int at    = r.target - first_class - col;
    const float g   = r.target < 0 ? NAN : r.grad;
    typedef T vec __attribute__((ext_vector_type(4)));
    vec out, rest;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float x = col + e < n ? (expFast(v[e] - r.lse) - (e == at ? 1.f : 0.f)) * g : 0.f;
        out[e]        = static_cast<T>(x);
        rest[e]       = static_cast<T>(x - toFloat(static_cast<T>(x)));
    }
    T* const to                 = dl + row * pair * ldd + col;
    *reinterpret_cast<vec*>(to) = out;
    if (pair == 2) *reinterpret_cast<vec*>(to + ldd) = rest;
}

// loss and lse of every kept token from its parts' maxima and sums, 0 of the others.  A workgroup takes 16
// tokens, 64 threads each: a quarter of a wave loads adjacent tokens, a thread every 64th part, four loads
// in flight.  (64 tokens, a wave's lanes each one, eight in flight: 6.6 us for 16 tokens of 251 parts, 4.7 so.)
// place: null without packing.
constexpr int kFinishTokens = 16;
__global__ __launch_bounds__(kFinishThreads) void finishLoss(const float2* part, const float* hit, Targets targets,
                                                             const int32_t* place, int64_t tokens, int parts, float* loss,
                                                             float* lse) {
    constexpr int kWaves = kFinishThreads / kWave, kShare = kFinishThreads / kFinishTokens, kBatch = 4;
    static_assert(kWave / kFinishTokens == 4 && kWaves == 4 * kBatch, "four threads a token in a wave, which join the waves");
    __shared__ float2 met[kWaves][kFinishTokens];
    const int token = threadIdx.x % kFinishTokens, share = threadIdx.x / kFinishTokens;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kFinishTokens + token;
    int64_t row     = -1;
    if (t < tokens) row = place != nullptr ? place[t] : targets.given(t) != targets.ignore_index ? t : -1;
    float top = -INFINITY, sum = 0.f;
    // (top, sum) and v's joined; minus infinity has no sum.
    auto join = [&](auto& v) {
        float high = top;
        for (const float2& x : v) high = fmaxf(high, x.x);
        const float base = high == -INFINITY ? 0.f : high;
        sum *= expf(top - base);
        for (const float2& x : v) sum += x.y * expf(x.x - base);
        top = high;
    };
    auto joinLanes = [&] {
#pragma unroll
        for (int d = kFinishTokens; d < kWave; d <<= 1) {
            float2 v[1] = {make_float2(__shfl_xor(top, d, kWave), __shfl_xor(sum, d, kWave))};
            join(v);
        }
    };
    // Asked for with the parts.
    const bool last = share == 0 && row >= 0;
    const int y     = last ? targets(row) : -1;
    const float l_y = y >= 0 ? hit[row] : 0.f;
    if (row >= 0) {
        for (int i = share; i < parts; i += kShare * kBatch) {
            float2 v[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                v[b] = i + b * kShare < parts ? part[(i + b * kShare) * tokens + row] : make_float2(-INFINITY, 0.f);
            join(v);
        }
    }
    joinLanes();
    if (threadIdx.x % kWave < kFinishTokens) met[threadIdx.x / kWave][token] = make_float2(top, sum);
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    float2 v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) v[b] = met[share * kBatch + b][token];
    top = -INFINITY, sum = 0.f;
    join(v);
    joinLanes();
    if (share != 0 || t >= tokens) return;
    // Not lse - l_y: where the target holds nearly all, the loss is far smaller than the rounding of lse.
    const float log_sum = logf(sum);
    lse[t]              = row < 0 ? 0.f : top + log_sum;
    loss[t]             = row < 0 ? 0.f : y < 0 ? NAN : (top - l_y) + log_sum;
}

// grad_hidden row t: the packed row's sums, rounded once; zeros for an ignored token.  A lane takes four
// columns.  MANY: the workgroup's waves share the slices of 256 columns, joined in LDS (16 tokens of 4096
// in 62 slices of two rows: 60 -> 4.8 us), else they take columns of their own.
template <class T, bool MANY>
__global__ __launch_bounds__(kThreads) void finishHidden(const float* sums, int64_t ld, const int32_t* place,
                                                         const Head* head, T* out, int64_t out_ld, int64_t tokens,
                                                         int64_t cols, int slices, int64_t slice, int pair) {
    constexpr int kWaves = kThreads / kWave;
    __shared__ float4 met[MANY ? kWaves : 1][kWave];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const float inv = head->inv_scale;
    const int64_t i = MANY ? static_cast<int64_t>(blockIdx.y) * (4 * kWave) + 4 * lane
                           : (static_cast<int64_t>(blockIdx.y) * kThreads + threadIdx.x) * 4;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
        const int row = place[t];
        float4 v      = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row >= 0 && i < cols) {
            const float* const from = sums + static_cast<int64_t>(row) * pair * ld + i;
            v = sumSlices(MANY ? wave : 0, MANY ? kWaves : 1, slices * pair,
                          [&](int z) { return from + (pair == 2 ? (z >> 1) * slice + (z & 1) * ld : z * slice); });
        }
        if constexpr (MANY) {
            __syncthreads();
            met[wave][lane] = v;
            __syncthreads();
            if (wave != 0) continue;
            for (int w = 1; w < kWaves; ++w) {
                const float4 x = met[w][lane];
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
        }
        if (i >= cols) continue;
        T* const to = out + t * out_ld + i;
        to[0]       = static_cast<T>(v.x * inv);
        if (i + 1 < cols) to[1] = static_cast<T>(v.y * inv);
        if (i + 2 < cols) to[2] = static_cast<T>(v.z * inv);
        if (i + 3 < cols) to[3] = static_cast<T>(v.w * inv);
    }
}

uint64_t ceilDiv(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
uint64_t roundUp(uint64_t a, uint64_t b) { return ceilDiv(a, b) * b; }

// Bytes of a piece of dl.  Small pieces fill the device badly and add dx up more often; 8192 x 4096 x
// 131072 (16384 x 2048 x 65536) bf16 gradients, us, at 64 MiB 18494 (13042), 128 17655 (10997), 256 17507
// (9380), 512 17371 (9234), 1024 17256 (9204).
constexpr uint64_t kPieceBytes = 512ull << 20;
constexpr uint64_t kCus = 256;

// How a product runs: tile rows (launchHeadTile), and slices of k that keep sums of their own.
struct Tiling {
    int rows;
    int slices;
    double micros;  // modelled
};

// Modelled time of an m x n x k product, us: rounds of the 256 CUs, each of its stages and a start and
// end.  Measured per stage: 16-bit (64 k) 256x256 1.25 (0.75 with at most 128 rows), 128x128 0.5, 64x128 0.3;
// fp32 (32 k) 128x128 1.75, 64x64 0.5.  A large tile reads less for each product, a small one fills the CUs
// where there are few:
//   bf16, us, 256x256 / 128x128: loss of 128 x 1024 x 8192 27.8 / 24.0, 500 x 1024 x 5003 40.5 / 23.2,
//     64 x 4096 x 128000 201 / 234; gradients of 500 x 1024 x 5003 77.6 / 60.2, 2048 x 4096 x 32003
//     1198 / 1392;
//   fp32, us, 128x128 / 64x64: loss of 300 x 8192 x 3000 470 / 166, 1000 x 1000 x 1000 80 / 36.
double tileMicros(bool fp32, HeadTile what, int rows, int cols, int64_t m, int64_t n, int64_t k, int slices) {
    // dw's 128x128 tiles run two to a CU: fp16 500 x 1024 x 5003 15.5 us against 16.4 on 256x256, bf16
    // 200 x 4096 x 10000 47.9 against 41.5, 16 x 4096 x 32003 113 against 80.
    if (what == HeadTile::kGradWeight && rows == 128)
        return static_cast<double>(ceilDiv(ceilDiv(m, rows) * ceilDiv(n, cols), 2 * kCus)) * (static_cast<double>(k) / 64 * 0.8 + 10.0);
    const uint64_t tiles = ceilDiv(m, rows) * ceilDiv(n, cols) * slices;
    // The 64x128 tile runs two to a CU; loss (gradients) with 128x128 / 64x128 of 65 x 512 x 1000 bf16 15.6 /
    // 13.1 (26.2 / 24.2), 256 x 256 x 256 14.7 / 12.7 (20.2 / 18.0), 200 x 4096 x 10000 41.2 / 47.7 (117 / 121),
    // 700 x 2048 x 4000 30.4 / 32.7 (76 / 78), 1000 x 1024 x 8000 36.3 / 35.5 (97.5 / 91.7).
    const bool twice = !fp32 && rows == 64 && tiles > kCus;
    const double stage = fp32 ? (rows == 128 ? 1.75 : 0.5)
                         : rows == 256 ? (m <= 128 ? 0.75 : 1.25)
                         : rows == 128 ? 0.5
                                       : (twice ? 0.58 : 0.3);
    const double ends = fp32 ? 5.0 : rows == 256 ? 9.0 : rows == 128 && what == HeadTile::kGradLogits ? 8.0 : 6.0;
    const uint64_t rounds = ceilDiv(tiles, (twice ? 2 : 1) * kCus);
    return static_cast<double>(rounds) * (static_cast<double>(ceilDiv(k, slices)) / (fp32 ? 32 : 64) * stage + ends);
}

// Most bytes of the logits' slices, and what a further launch to join them takes, us.
constexpr uint64_t kSliceBytes = 64ull << 20;
constexpr double kJoinMicros   = 5.0;

// k may be cut, in slices of at least 512, until the tiles fill the device (two workgroups of fp32 and of
// the 64x128 tile run on a CU): dx's always, as its sums are fp32 in the workspace anyway; the logits'
// where few tokens' few tiles have a long k, at the price of writing and reading the slices (at 4 TB/s)
// and a launch: gradients of 16 x 8192 x 4000 fp32 255 -> 146 us; also where a last round is nearly
// empty, loss of 16 x 8192 x 20000 fp32 274 -> 198.  (With 200 x 4096 x 10000 8% of
// 528 us: not done.)
Tiling tilingOf(FTrainNumericType type, HeadTile what, int64_t m, int64_t n, int64_t k) {
    const bool fp32 = type == FTRAIN_NUMERIC_TYPE_FP32, hidden = what == HeadTile::kGradHidden;
    // The rows of the weight's gradient are the classes: many, and fp32 has the large tile only.
    if (fp32 && what == HeadTile::kGradWeight) return {128, 1, 0.0};
    Tiling best{};
    auto consider = [&](int rows, int cols, int at_once) {
        const uint64_t tiles = std::max<uint64_t>(1, ceilDiv(m, rows) * ceilDiv(n, cols));
        const int most       = static_cast<int>(std::max<uint64_t>(1, std::min<uint64_t>(at_once * kCus / tiles, k / 512)));
        auto offer           = [&](int slices, double more) {
            const double micros = tileMicros(fp32, what, rows, cols, m, n, k, slices) + more;
            if (best.rows == 0 || micros < best.micros) best = {rows, slices, micros};
        };
        if (hidden) {
            offer(most, 0.0);
            return;
        }
        offer(1, 0.0);
        if (what == HeadTile::kGradWeight || m > kFewTokens) return;
        for (int slices = 2; slices <= std::min<int64_t>(std::max(most, 8), k / 512); ++slices) {
            const double bytes = 4.0 * m * roundUp(n, 256) * slices;
            if (bytes <= kSliceBytes) offer(slices, kJoinMicros + 2.0 * bytes / 4e6);
        }
    };
    if (!fp32 && what != HeadTile::kGradWeight && m <= kFewTokens) {
        consider(64, 128, 2);
    } else {
        consider(fp32 ? 128 : 256, fp32 ? 128 : 256, fp32 ? 2 : 1);
        consider(fp32 ? 64 : 128, fp32 ? 64 : 128, fp32 ? 2 : 1);
        if (!fp32 && !hidden && what != HeadTile::kGradWeight) consider(64, 128, 2);
    }
    return best;
}

// Row strides from which 64 rows are 2^30 bytes: the tiles' offsets are 32 bits.
constexpr int64_t kDirectLd = int64_t(1) << 22;

// The workspace, laid out for one call.
struct Layout {
    uint64_t bytes = 0;
    uint64_t head, place, rows, x, w, part, hit, cut, dl, dx;
    int64_t padded;  // columns of a packed row of x (and w)
    int64_t piece;   // classes of one piece
    int64_t pair;    // rows of x and dl of each token (kFewTokens)
    // The loss of few tokens, x in whole 16-byte units: no packing (the smallest tile holds every token;
    // what an ignored one is worth stays in its row).  16 x 4096 x 32003 bf16 57.8 -> 51.8 us.
    bool direct;
    int64_t parts;
    Tiling logits, for_hidden, for_weight;
    int64_t cut_ld;  // row stride of the logits' slices, where k is cut
    int64_t slice;   // elements of one slice's sums
    bool joint;      // dx and dw in one launch
    bool pack_w;     // the weight's rows are not whole 16-byte units: each piece is copied first

    Layout(const CrossEntropy& p, bool backward) {
        const uint64_t tokens = p.hidden.rows, hidden = p.hidden.cols, classes = p.weight.rows;
        const uint64_t size = elementBytes(p.type), unit = 16 / size;
        pair   = backward && size == 2 && tokens <= kFewTokens ? 2 : 1;
        padded = roundUp(hidden, unit);
        pack_w = hidden % unit != 0 || p.weight.ld % unit != 0 || reinterpret_cast<uintptr_t>(p.weight.data) % 16 != 0;
        direct = !backward && static_cast<int64_t>(tokens) <= kFewTokens && hidden % unit == 0 && p.hidden.ld % unit == 0 &&
                 p.hidden.ld < kDirectLd && reinterpret_cast<uintptr_t>(p.hidden.data) % 16 == 0;
        const uint64_t row = backward ? pair * tokens * size : pack_w ? padded * size : 1;
        piece = std::min(std::max<uint64_t>(kPieceBytes / std::max<uint64_t>(row, 1) / 256 * 256, 2048), roundUp(classes, 256));
        const int64_t n = backward || pack_w ? std::min<int64_t>(piece, classes) : classes;
        logits = tilingOf(p.type, backward ? HeadTile::kGradLogits : HeadTile::kLogSum, tokens, n, padded);
        // Classes of one part: a 16-bit tile's columns, the 64 that an fp32 wave holds, or joinLogSum's.
        parts      = ceilDiv(classes, logits.slices > 1               ? 256
                                      : p.type == FTRAIN_NUMERIC_TYPE_FP32 ? 64
                                      : logits.rows == 256                 ? 256
                                                                           : 128);
        cut_ld     = roundUp(n, 256);
        for_hidden = tilingOf(p.type, HeadTile::kGradHidden, pair * tokens, hidden, n);
        for_weight = tilingOf(p.type, HeadTile::kGradWeight, n, hidden, pair * tokens);
        joint      = size == 2 && tokens > 0 && joinGradients(pair * tokens, n, padded);
        slice     = pair * tokens * padded;
        auto take = [&](uint64_t n) {
            const uint64_t at = bytes;
            bytes += roundUp(n, 256);
            return at;
        };
        head  = take(sizeof(Head));
        place = take(tokens * 4);
        rows  = take(tokens * sizeof(RowInfo));
        x     = take(direct ? 0 : pair * tokens * padded * size);
        w     = pack_w ? take(piece * padded * size) : 0;
        part  = backward ? 0 : take(tokens * parts * sizeof(float2));
        hit   = backward ? 0 : take(tokens * 4);
        cut   = logits.slices > 1 ? take(logits.slices * tokens * cut_ld * 4) : 0;
        dl    = backward ? take(pair * tokens * piece * size) : 0;
        dx    = backward ? take(for_hidden.slices * slice * 4) : 0;
    }

  private:
    // Both products of dl, 16-bit, in one launch of 128x128 tiles, two workgroups to a CU: dx's slices fill
    // the rounds that dw's tiles begin.  us in two launches and in one: 500 x 1024 x 5003 fp16 gradients
    // 52.9 / 46.3, 2000 x 512 x 3000 bf16 72.3 / 62.9, 65 x 512 x 1000 35.1 / 26.2, 256 x 256 x 256 25.3 / 20.2.
    bool joinGradients(uint64_t m, uint64_t n, uint64_t hidden) {
        const uint64_t cols   = ceilDiv(hidden, 128), begun = ceilDiv(n, 128) * cols;
        const uint64_t tiles  = std::max<uint64_t>(1, ceilDiv(m, 128) * cols);
        const uint64_t round  = 2 * kCus, room = roundUp(begun + tiles, round) - begun;
        const uint64_t slices = std::max<uint64_t>(1, std::min<uint64_t>(room / tiles, n / 512));
        const double stages   = static_cast<double>(std::max(m, ceilDiv(n, slices))) / 64;
        const double micros   = static_cast<double>(ceilDiv(begun + tiles * slices, round)) * (stages * 0.8 + 10.0);
        if (micros >= for_hidden.micros + for_weight.micros) return false;
        for_hidden = {128, static_cast<int>(slices), micros};
        for_weight = {128, 1, micros};
        return true;
    }
};

struct Buffers {
    Head* head;
    int32_t* place;
    RowInfo* rows;
    char* base;
};

Targets targetsOf(const CrossEntropy& p, const RowInfo* rows) {
    return Targets{rows, p.target, p.ignore_index, p.weight.rows, p.target_wide};
}

template <class T>
Buffers packInputs(const CrossEntropy& p, const Layout& l, char* base, bool backward, hipStream_t stream) {
    Buffers b{reinterpret_cast<Head*>(base + l.head), reinterpret_cast<int32_t*>(base + l.place),
              reinterpret_cast<RowInfo*>(base + l.rows), base};
    PackArgs a{};
    a.targets = targetsOf(p, nullptr), a.tokens = p.hidden.rows;
    a.lse = p.lse, a.grad_loss = p.grad_loss;
    a.head = b.head, a.place = b.place, a.rows = b.rows;
    a.x = p.hidden.data, a.ld = p.hidden.ld, a.cols = p.hidden.cols;
    a.packed = base + l.x, a.padded = l.padded, a.pair = static_cast<int>(l.pair);
    a.backward = backward, a.scaled = backward && p.type == FTRAIN_NUMERIC_TYPE_FP16;
    a.per_block        = std::max<int64_t>(1, ceilDiv(a.tokens, kPackBlocks));
    const int64_t grid = std::max<int64_t>(1, ceilDiv(a.tokens, a.per_block));
    launch(&packTokens<T>, "cross entropy pack", dim3(static_cast<uint32_t>(grid)), dim3(kPackThreads), stream, a);
    return b;
}

void launchHeadTile(FTrainNumericType type, HeadTile what, int rows, const HeadTileArgs& args, int slices, hipStream_t stream) {
    if (type == FTRAIN_NUMERIC_TYPE_FP32)
        launchHeadTileFp32(what, rows, args, slices, stream);
    else if (type == FTRAIN_NUMERIC_TYPE_BF16)
        launchHeadTileBf16(what, rows, args, slices, stream);
    else
        launchHeadTileFp16(what, rows, args, slices, stream);
}

// The classes from `first` on, `n` of them, in rows of whole 16-byte units.
template <class T>
const T* weightPiece(const CrossEntropy& p, const Layout& l, char* base, int64_t first, int64_t n, int64_t& ld,
                     hipStream_t stream) {
    const T* const from = static_cast<const T*>(p.weight.data) + first * p.weight.ld;
    ld                  = p.weight.ld;
    if (!l.pack_w) return from;
    T* const to = reinterpret_cast<T*>(base + l.w);
    launch(&packWeight<T>, "cross entropy weight pack", dim3(static_cast<uint32_t>(std::min<int64_t>(ceilDiv(n, 4), 4096))),
           dim3(kThreads), stream, from, p.weight.ld, n, p.weight.cols, to, l.padded);
    ld = l.padded;
    return to;
}

// The logits' slices of the classes that t describes.
void cutLogits(const CrossEntropy& p, const Layout& l, char* base, HeadTileArgs t, hipStream_t stream) {
    t.d = base + l.cut, t.ldd = l.cut_ld, t.slice = p.hidden.rows * l.cut_ld;
    t.k_chunk = roundUp(ceilDiv(t.k, l.logits.slices), 64);
    launchHeadTile(p.type, HeadTile::kLogits, l.logits.rows, t, l.logits.slices, stream);
}
dim3 joinGrid(int64_t tokens, int64_t n) {
    return dim3(static_cast<uint32_t>(ceilDiv(n, 256)), static_cast<uint32_t>(ceilDiv(tokens, kThreads / kWave)));
}

template <class T>
void forward(const CrossEntropy& p, char* base, hipStream_t stream) {
    const Layout l(p, false);
    const Buffers b = l.direct ? Buffers{} : packInputs<T>(p, l, base, false, stream);
    HeadTileArgs t{};
    t.a   = l.direct ? p.hidden.data : base + l.x;
    t.lda = l.direct ? p.hidden.ld : l.padded;
    t.m = p.hidden.rows, t.k = l.padded;
    t.head = b.head, t.targets = targetsOf(p, b.rows);
    t.part = reinterpret_cast<float2*>(base + l.part), t.hit = reinterpret_cast<float*>(base + l.hit);
    t.tokens              = p.hidden.rows;
    const int64_t classes = p.weight.rows, piece = l.pack_w ? l.piece : classes;
    for (int64_t v = 0; v < classes; v += piece) {
        t.n = std::min(piece, classes - v), t.first_class = v;
        t.b = weightPiece<T>(p, l, base, v, t.n, t.ldb, stream);
        if (l.logits.slices == 1) {
            launchHeadTile(p.type, HeadTile::kLogSum, l.logits.rows, t, 1, stream);
            continue;
        }
        cutLogits(p, l, base, t, stream);
        launch(&joinLogSum, "cross entropy join", joinGrid(t.m, t.n), dim3(kThreads), stream,
               reinterpret_cast<const float*>(base + l.cut), l.cut_ld, t.m * l.cut_ld, l.logits.slices,
               static_cast<const Head*>(b.head), t.targets, t.n, t.first_class, t.tokens, t.part, t.hit);
    }
    launch(&finishLoss, "cross entropy loss", dim3(static_cast<uint32_t>(ceilDiv(p.hidden.rows, kFinishTokens))),
           dim3(kFinishThreads), stream, static_cast<const float2*>(t.part), static_cast<const float*>(t.hit),
           t.targets, static_cast<const int32_t*>(b.place), p.hidden.rows, static_cast<int>(l.parts), p.loss, p.lse);
}

template <class T>
void backward(const CrossEntropy& p, char* base, hipStream_t stream) {
    const Layout l(p, true);
    const Buffers b = packInputs<T>(p, l, base, true, stream);
    const int64_t tokens = p.hidden.rows, hidden = p.hidden.cols, classes = p.weight.rows;
    const int64_t unit = 16 / sizeof(T);
    for (int64_t v = 0; v < classes; v += l.piece) {
        HeadTileArgs t{};
        t.head = b.head, t.targets = targetsOf(p, b.rows), t.first_class = v, t.pair = static_cast<int32_t>(l.pair);
        const int64_t n = std::min(l.piece, classes - v);
        int64_t ldw;
        const T* const w = weightPiece<T>(p, l, base, v, n, ldw, stream);
        HeadTileArgs of_x = t, of_w = t;
        int slices = 0;
        if (tokens > 0) {
            t.a = base + l.x, t.lda = l.pair * l.padded;
            t.b = w, t.ldb = ldw;
            t.d = base + l.dl, t.ldd = l.piece;
            t.m = tokens, t.n = n, t.k = l.padded;
            if (l.logits.slices == 1) {
                launchHeadTile(p.type, HeadTile::kGradLogits, l.logits.rows, t, 1, stream);
            } else {
                cutLogits(p, l, base, t, stream);
                launch(&joinGradLogits<T>, "cross entropy join", joinGrid(tokens, n), dim3(kThreads), stream,
                       reinterpret_cast<const float*>(base + l.cut), l.cut_ld, tokens * l.cut_ld, l.logits.slices,
                       static_cast<const Head*>(b.head), static_cast<const RowInfo*>(b.rows), t.n,
                       static_cast<int>(roundUp(n, unit)), t.first_class, reinterpret_cast<T*>(base + l.dl), l.piece,
                       static_cast<int>(l.pair));
            }
            of_x.a = base + l.dl, of_x.lda = l.piece;
            of_x.b = w, of_x.ldb = ldw;
            of_x.d = base + l.dx, of_x.ldd = l.padded;
            of_x.m = l.pair * tokens, of_x.n = l.padded, of_x.k = n;
            // Whole stages of the tile to a slice; a last piece's slices may be fewer, its sums then
            // leave the others as they are.
            of_x.k_chunk = roundUp(ceilDiv(n, l.for_hidden.slices), 64);
            of_x.slice   = l.slice;
            of_x.add     = v > 0;
            slices       = of_x.add ? static_cast<int>(ceilDiv(n, of_x.k_chunk)) : l.for_hidden.slices;
        }
        of_w.a = base + l.dl, of_w.lda = l.piece;
        of_w.b = base + l.x, of_w.ldb = l.padded;
        of_w.d = static_cast<T*>(p.grad_weight.data) + v * p.grad_weight.ld, of_w.ldd = p.grad_weight.ld;
        of_w.m = n, of_w.n = hidden, of_w.k = l.pair * tokens;
        of_w.read_m = roundUp(n, unit), of_w.read_n = l.padded;
        if (l.joint) {
            (p.type == FTRAIN_NUMERIC_TYPE_BF16 ? launchHeadGradientsBf16 : launchHeadGradientsFp16)(of_x, slices, of_w, stream);
            continue;
        }
        if (tokens > 0) launchHeadTile(p.type, HeadTile::kGradHidden, l.for_hidden.rows, of_x, slices, stream);
        launchHeadTile(p.type, HeadTile::kGradWeight, l.for_weight.rows, of_w, 1, stream);
    }
    if (tokens == 0) return;
    const bool many = l.for_hidden.slices * l.pair >= 8;
    launch(many ? &finishHidden<T, true> : &finishHidden<T, false>, "cross entropy hidden gradient's rows",
           dim3(static_cast<uint32_t>(std::min<int64_t>(tokens, 65536)),
                static_cast<uint32_t>(ceilDiv(hidden, many ? 4 * kWave : 4 * kThreads))),
           dim3(kThreads), stream, reinterpret_cast<const float*>(base + l.dx), l.padded, static_cast<const int32_t*>(b.place),
           static_cast<const Head*>(b.head), static_cast<T*>(p.grad_hidden.data), p.grad_hidden.ld, tokens, hidden,
           l.for_hidden.slices, l.slice, static_cast<int>(l.pair));
}

}  // namespace

uint64_t crossEntropyWorkspace(const CrossEntropy& p, bool backward) { return Layout(p, backward).bytes; }

void crossEntropyForward(const CrossEntropy& p, void* workspace, hipStream_t stream) {
    if (p.hidden.rows == 0) return;
    char* const base = static_cast<char*>(workspace);
    if (p.type == FTRAIN_NUMERIC_TYPE_FP32)
        forward<float>(p, base, stream);
    else if (p.type == FTRAIN_NUMERIC_TYPE_BF16)
        forward<bf16>(p, base, stream);
    else
        forward<fp16>(p, base, stream);
}

void crossEntropyBackward(const CrossEntropy& p, void* workspace, hipStream_t stream) {
    char* const base = static_cast<char*>(workspace);
    if (p.type == FTRAIN_NUMERIC_TYPE_FP32)
        backward<float>(p, base, stream);
    else if (p.type == FTRAIN_NUMERIC_TYPE_BF16)
        backward<bf16>(p, base, stream);
    else
        backward<fp16>(p, base, stream);
}

}  // namespace ftrain::train
