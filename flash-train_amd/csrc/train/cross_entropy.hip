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
// and how it is aligned is thereby settled too.  A target outside the classes makes its token's loss
// and gradients NaN.
#include <algorithm>

#include "device.hpp"
#include "ft/train.hpp"

namespace ftrain::train {
namespace {

constexpr int kThreads     = 256;
constexpr int kPackThreads = 1024;

// What the device knows of the batch.
struct Head {
    int32_t valid;    // packed rows
    float scale;      // dl is kept times this power of two
    float inv_scale;
};

// One packed row: where its gradient of the loss, its lse and its target are.
struct RowInfo {
    float lse;
    float grad;      // times Head::scale
    int32_t target;  // -1: outside the classes
};

struct PackArgs {
    const void* target;
    int64_t ignore_index;
    int64_t tokens, classes;
    float *loss, *lse;       // forward: 0 where ignored
    const float* grad_loss;  // backward
    Head* head;
    int32_t* place;  // each token's packed row, -1 if ignored
    RowInfo* rows;
    bool wide, backward, scaled;
};

// One workgroup: each token's packed row, in order.
__global__ __launch_bounds__(kPackThreads) void packRows(PackArgs a) {
    constexpr int kWaves = kPackThreads / kWave;
    __shared__ int wave_count[kWaves];
    __shared__ float wave_max[kWaves];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    auto target = [&](int64_t t) {
        return a.wide ? static_cast<const int64_t*>(a.target)[t]
                      : static_cast<int64_t>(static_cast<const int32_t*>(a.target)[t]);
    };
    float scale = 1.f;
    if (a.scaled) {
        // fp16 holds no small probability: dl is kept times the power of two that brings the largest
        // |g| into [2^14, 2^15), |dl| <= |g| stays below fp16's largest value, and what is lost is
        // below 2^-39 of the largest g.
        float top = 0.f;
        for (int64_t t = threadIdx.x; t < a.tokens; t += kPackThreads)
            if (target(t) != a.ignore_index) top = fmaxf(top, fabsf(a.grad_loss[t]));
        top = groupMax<kWave>(top);
        if (lane == 0) wave_max[wave] = top;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_max[w]);
        if (top > 0.f && top < INFINITY) {
            int e;
            (void)frexpf(top, &e);  // top in [2^(e-1), 2^e)
            scale = ldexpf(1.f, min(15 - e, 120));
        }
    }
    int before = 0;
    for (int64_t t0 = 0; t0 < a.tokens; t0 += kPackThreads) {
        const int64_t t  = t0 + threadIdx.x;
        const int64_t y  = t < a.tokens ? target(t) : a.ignore_index;
        const bool kept  = t < a.tokens && y != a.ignore_index;
        const unsigned long long mask = __ballot(kept);
        if (lane == 0) wave_count[wave] = __popcll(mask);
        __syncthreads();
        int at = before + __popcll(mask & ((1ull << lane) - 1ull));
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) at += wave_count[w];
            before += wave_count[w];
        }
        __syncthreads();
        if (t < a.tokens) {
            a.place[t] = kept ? at : -1;
            if (kept)
                a.rows[at] = RowInfo{a.backward ? a.lse[t] : 0.f, a.backward ? a.grad_loss[t] * scale : 0.f,
                                     y >= 0 && y < a.classes ? static_cast<int32_t>(y) : -1};
            else if (!a.backward)
                a.loss[t] = a.lse[t] = 0.f;
        }
    }
    if (threadIdx.x == 0) *a.head = Head{before, scale, 1.f / scale};
}

// dst row place[t] (row t with a null place) = src row t, padded with zeros to `padded` columns.
template <class T>
__global__ __launch_bounds__(kThreads) void copyRows(const T* src, int64_t src_ld, int64_t rows, int64_t cols, T* dst,
                                                     int64_t dst_ld, int64_t padded, const int32_t* place) {
    for (int64_t t = blockIdx.x; t < rows; t += gridDim.x) {
        const int64_t to = place != nullptr ? place[t] : t;
        if (to < 0) continue;
        const T* const from = src + t * src_ld;
        T* const out        = dst + to * dst_ld;
        constexpr int N     = Pack<T>::kCount;
        const int64_t whole = cols / N * N;
        for (int64_t i = threadIdx.x * N; i < whole; i += kThreads * N)
            *reinterpret_cast<Pack<T>*>(out + i) = *reinterpret_cast<const Pack<T>*>(from + i);
        for (int64_t i = whole + threadIdx.x; i < padded; i += kThreads) out[i] = i < cols ? from[i] : static_cast<T>(0.f);
    }
}

enum class Mode { kLogSum, kGradLogits, kGradHidden, kGradWeight };

struct TileArgs {
    const void *a, *b;  // element (i, k) of a at i a_row + k a_col, (k, j) of b at k b_row + j b_col
    int64_t a_row, a_col, b_row, b_col;
    int32_t m, n, k;
    const Head* head;
    const RowInfo* rows;
    int32_t first_class;
    float2* part;  // kLogSum: of each row, each tile column's maximum and sum
    float* hit;    // kLogSum: each row's logit of its target
    int32_t parts;
    void* d;
    int64_t ldd;
    int32_t padded;  // kGradLogits: columns to write (zeros past n)
    bool add;        // kGradHidden
};

// A 64x64 tile of a @ b by 256 threads, 4x4 outputs each, and what the mode makes of it.
template <class T, Mode MODE>
__global__ __launch_bounds__(kThreads) void tile(TileArgs p) {
    constexpr int S = 64, K = 16;
    __shared__ float As[K][S + 4], Bs[K][S + 4];
    const int valid = p.head->valid;
    const int M = MODE == Mode::kGradWeight ? p.m : min(p.m, valid), N = p.n;
    const int D = MODE == Mode::kGradWeight ? min(p.k, valid) : p.k;
    const int m0 = blockIdx.y * S, n0 = blockIdx.x * S;
    if (m0 >= M) return;
    const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    const T* const a = static_cast<const T*>(p.a);
    const T* const b = static_cast<const T*>(p.b);
    float acc[4][4] = {};
    for (int k0 = 0; k0 < D; k0 += K) {
        for (int i = threadIdx.x; i < S * K; i += kThreads) {
            const int ak = p.a_col == 1 ? i % K : i / S, am = p.a_col == 1 ? i / K : i % S;
            As[ak][am] = m0 + am < M && k0 + ak < D ? toFloat(a[(m0 + am) * p.a_row + (k0 + ak) * p.a_col]) : 0.f;
            const int bk = p.b_row == 1 ? i % K : i / S, bn = p.b_row == 1 ? i / K : i % S;
            Bs[bk][bn] = n0 + bn < N && k0 + bk < D ? toFloat(b[(k0 + bk) * p.b_row + (n0 + bn) * p.b_col]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[k][4 * tr + i], Bs[k][4 * tc + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
        const int row = m0 + 4 * tr + i;
        if constexpr (MODE == Mode::kLogSum) {
            float top = -INFINITY, sum = 0.f;
            const int y = row < M ? p.rows[row].target - p.first_class : -1;
            for (int j = 0; j < 4; ++j) {
                const int col = n0 + 4 * tc + j;
                if (col < N) top = fmaxf(top, acc[i][j]);
                if (row < M && col < N && col == y) p.hit[row] = acc[i][j];
            }
            top = groupMax<16>(top);
            for (int j = 0; j < 4; ++j)
                if (n0 + 4 * tc + j < N) sum += expf(acc[i][j] - top);
            sum = groupSum<16>(sum);
            if (tc == 0 && row < M)
                p.part[static_cast<int64_t>(row) * p.parts + p.first_class / S + blockIdx.x] = make_float2(top, sum);
        } else if (row < M) {
            for (int j = 0; j < 4; ++j) {
                const int col = n0 + 4 * tc + j;
                if constexpr (MODE == Mode::kGradLogits) {
                    if (col >= p.padded) continue;
                    const RowInfo r = p.rows[row];
                    float v         = 0.f;
                    if (col < N) {
                        v = expf(acc[i][j] - r.lse) - (col == r.target - p.first_class ? 1.f : 0.f);
                        v = r.target < 0 ? NAN : v * r.grad;
                    }
                    static_cast<T*>(p.d)[row * p.ldd + col] = static_cast<T>(v);
                } else if (col < N) {
                    if constexpr (MODE == Mode::kGradHidden) {
                        float* const d = static_cast<float*>(p.d) + row * p.ldd + col;
                        *d             = p.add ? *d + acc[i][j] : acc[i][j];
                    } else {
                        static_cast<T*>(p.d)[row * p.ldd + col] = static_cast<T>(acc[i][j] * p.head->inv_scale);
                    }
                }
            }
        }
    }
}

// loss and lse of every kept token from its tiles' maxima and sums; a wave per token.
__global__ __launch_bounds__(kThreads) void finishLoss(const float2* part, const float* hit, const RowInfo* rows,
                                                       const int32_t* place, int64_t tokens, int parts, float* loss,
                                                       float* lse) {
    const int lane  = threadIdx.x % kWave;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + threadIdx.x / kWave;
    if (t >= tokens) return;
    const int row = place[t];
    if (row < 0) return;
    const float2* const mine = part + static_cast<int64_t>(row) * parts;
    float top = -INFINITY;
    for (int i = lane; i < parts; i += kWave) top = fmaxf(top, mine[i].x);
    top = groupMax<kWave>(top);
    float sum = 0.f;
    for (int i = lane; i < parts; i += kWave) {
        const float2 v = mine[i];
        // A tile of nothing but minus infinity has no sum.
        sum += v.x == -INFINITY && top > -INFINITY ? 0.f : v.y * expf(v.x - top);
    }
    sum = groupSum<kWave>(sum);
    if (lane == 0) {
        const float l = top + logf(sum);
        lse[t]        = l;
        loss[t]       = rows[row].target < 0 ? NAN : l - hit[row];
    }
}

// grad_hidden row t: the packed row's sums, rounded once; zeros for an ignored token.
template <class T>
__global__ __launch_bounds__(kThreads) void finishHidden(const float* sums, int64_t ld, const int32_t* place,
                                                         const Head* head, T* out, int64_t out_ld, int64_t tokens,
                                                         int64_t cols) {
    const float inv = head->inv_scale;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
        const int row           = place[t];
        const float* const from = sums + static_cast<int64_t>(row) * ld;
        for (int64_t i = threadIdx.x; i < cols; i += kThreads)
            out[t * out_ld + i] = static_cast<T>(row < 0 ? 0.f : from[i] * inv);
    }
}

uint64_t ceilDiv(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
uint64_t roundUp(uint64_t a, uint64_t b) { return ceilDiv(a, b) * b; }

// The workspace, laid out for one call.
struct Layout {
    uint64_t bytes = 0;
    uint64_t head, place, rows, x, part, hit, dl, dx;
    int64_t padded;  // columns of a packed row of x
    int64_t piece;   // classes of one piece
    int64_t parts;

    Layout(const CrossEntropy& p, bool backward) {
        const uint64_t tokens = p.hidden.rows, hidden = p.hidden.cols, classes = p.weight.rows;
        const uint64_t size = elementBytes(p.type);
        padded              = roundUp(hidden, 16 / size);
        piece               = std::min<int64_t>(roundUp(classes, 64), 8192);
        parts               = ceilDiv(classes, 64);
        auto take           = [&](uint64_t n) {
            const uint64_t at = bytes;
            bytes += roundUp(n, 256);
            return at;
        };
        head  = take(sizeof(Head));
        place = take(tokens * 4);
        rows  = take(tokens * sizeof(RowInfo));
        x     = take(tokens * padded * size);
        part  = backward ? 0 : take(tokens * parts * sizeof(float2));
        hit   = backward ? 0 : take(tokens * 4);
        dl    = backward ? take(tokens * piece * size) : 0;
        dx    = backward ? take(tokens * padded * 4) : 0;
    }
};

struct Buffers {
    Head* head;
    int32_t* place;
    RowInfo* rows;
    char* base;
};

template <class T>
Buffers packInputs(const CrossEntropy& p, const Layout& l, char* base, bool backward, hipStream_t stream) {
    Buffers b{reinterpret_cast<Head*>(base + l.head), reinterpret_cast<int32_t*>(base + l.place),
              reinterpret_cast<RowInfo*>(base + l.rows), base};
    PackArgs a{p.target, p.ignore_index, p.hidden.rows, p.weight.rows, p.loss, p.lse, p.grad_loss, b.head,
               b.place,  b.rows,         p.target_wide, backward,      backward && p.type == FTRAIN_NUMERIC_TYPE_FP16};
    launch(&packRows, "cross entropy pack", dim3(1), dim3(kPackThreads), stream, a);
    if (p.hidden.rows > 0)
        launch(&copyRows<T>, "cross entropy copy", dim3(static_cast<uint32_t>(std::min<int64_t>(p.hidden.rows, 65536))),
           dim3(kThreads), stream, static_cast<const T*>(p.hidden.data), p.hidden.ld, p.hidden.rows, p.hidden.cols,
           reinterpret_cast<T*>(base + l.x), l.padded, l.padded, static_cast<const int32_t*>(b.place));
    return b;
}

dim3 gridOf(int64_t m, int64_t n) { return dim3(static_cast<uint32_t>(ceilDiv(n, 64)), static_cast<uint32_t>(ceilDiv(m, 64))); }

template <class T>
void forward(const CrossEntropy& p, char* base, hipStream_t stream) {
    const Layout l(p, false);
    const Buffers b = packInputs<T>(p, l, base, false, stream);
    TileArgs t{};
    t.a = base + l.x, t.a_row = l.padded, t.a_col = 1;
    t.b = p.weight.data, t.b_row = 1, t.b_col = p.weight.ld;
    t.m = p.hidden.rows, t.n = p.weight.rows, t.k = p.hidden.cols;
    t.head = b.head, t.rows = b.rows;
    t.part = reinterpret_cast<float2*>(base + l.part), t.hit = reinterpret_cast<float*>(base + l.hit);
    t.parts = l.parts;
    launch(&tile<T, Mode::kLogSum>, "cross entropy logits", gridOf(t.m, t.n), dim3(kThreads), stream, t);
    launch(&finishLoss, "cross entropy loss", dim3(static_cast<uint32_t>(ceilDiv(p.hidden.rows, kThreads / kWave))),
           dim3(kThreads), stream, static_cast<const float2*>(t.part), static_cast<const float*>(t.hit),
           static_cast<const RowInfo*>(b.rows), static_cast<const int32_t*>(b.place), p.hidden.rows,
           static_cast<int>(l.parts), p.loss, p.lse);
}

template <class T>
void backward(const CrossEntropy& p, char* base, hipStream_t stream) {
    const Layout l(p, true);
    const Buffers b = packInputs<T>(p, l, base, true, stream);
    const int64_t tokens = p.hidden.rows, hidden = p.hidden.cols, classes = p.weight.rows;
    for (int64_t v = 0; v < classes; v += l.piece) {
        const int64_t n  = std::min(l.piece, classes - v);
        const T* const w = static_cast<const T*>(p.weight.data) + v * p.weight.ld;
        TileArgs t{};
        t.head = b.head, t.rows = b.rows, t.first_class = v;
        t.a = base + l.x, t.a_row = l.padded, t.a_col = 1;
        t.b = w, t.b_row = 1, t.b_col = p.weight.ld;
        t.m = tokens, t.n = n, t.k = hidden;
        t.d = base + l.dl, t.ldd = l.piece, t.padded = n;
        if (tokens > 0) launch(&tile<T, Mode::kGradLogits>, "cross entropy logits' gradient", gridOf(tokens, n), dim3(kThreads), stream, t);
        t.a = base + l.dl, t.a_row = l.piece, t.a_col = 1;
        t.b = w, t.b_row = p.weight.ld, t.b_col = 1;
        t.n = hidden, t.k = n;
        t.d = base + l.dx, t.ldd = l.padded, t.add = v > 0;
        if (tokens > 0) launch(&tile<T, Mode::kGradHidden>, "cross entropy hidden gradient", gridOf(tokens, hidden), dim3(kThreads), stream, t);
        t.a_row = 1, t.a_col = l.piece;
        t.b = base + l.x, t.b_row = l.padded, t.b_col = 1;
        t.m = n, t.n = hidden, t.k = tokens;
        t.d = static_cast<T*>(p.grad_weight.data) + v * p.grad_weight.ld, t.ldd = p.grad_weight.ld;
        launch(&tile<T, Mode::kGradWeight>, "cross entropy weight gradient", gridOf(n, hidden), dim3(kThreads), stream, t);
    }
    if (tokens > 0) launch(&finishHidden<T>, "cross entropy hidden gradient's rows", dim3(static_cast<uint32_t>(std::min<int64_t>(tokens, 65536))),
           dim3(kThreads), stream, reinterpret_cast<const float*>(base + l.dx), l.padded,
           static_cast<const int32_t*>(b.place), static_cast<const Head*>(b.head), static_cast<T*>(p.grad_hidden.data),
           p.grad_hidden.ld, tokens, hidden);
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
