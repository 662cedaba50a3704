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

#include "cross_entropy.hpp"
#include "device.hpp"
#include "ft/train.hpp"

namespace ftrain::train {
namespace {

constexpr int kThreads     = 256;
constexpr int kPackThreads = 1024;

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
                                                         int64_t cols, int slices, int64_t slice) {
    const float inv = head->inv_scale;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
        const int row           = place[t];
        const float* const from = sums + static_cast<int64_t>(row) * ld;
        for (int64_t i = threadIdx.x * 4; i < cols; i += kThreads * 4) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row >= 0) {
                for (int z = 0; z < slices; ++z) {
                    const float4 x = *reinterpret_cast<const float4*>(from + z * slice + i);
                    v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
                }
            }
            T* const to = out + t * out_ld + i;
            to[0]       = static_cast<T>(v.x * inv);
            if (i + 1 < cols) to[1] = static_cast<T>(v.y * inv);
            if (i + 2 < cols) to[2] = static_cast<T>(v.z * inv);
            if (i + 3 < cols) to[3] = static_cast<T>(v.w * inv);
        }
    }
}

uint64_t ceilDiv(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
uint64_t roundUp(uint64_t a, uint64_t b) { return ceilDiv(a, b) * b; }

// Bytes of a piece of dl: the last-level cache's 256 MiB, which it is read from twice.
constexpr uint64_t kPieceBytes = 256ull << 20;
// Workgroups that fill the device's 256 CUs.
constexpr uint64_t kFill = 256;

// The workspace, laid out for one call.
struct Layout {
    uint64_t bytes = 0;
    uint64_t head, place, rows, x, w, part, hit, dl, dx;
    int64_t padded;  // columns of a packed row of x (and w)
    int64_t piece;   // classes of one piece
    int64_t parts;
    int slices;      // of a piece's classes, each with sums of its own for dx
    int64_t slice;   // elements of one slice's sums
    bool pack_w;     // the weight's rows are not whole 16-byte units: each piece is copied first

    Layout(const CrossEntropy& p, bool backward) {
        const uint64_t tokens = p.hidden.rows, hidden = p.hidden.cols, classes = p.weight.rows;
        const uint64_t size = elementBytes(p.type), unit = 16 / size;
        padded = roundUp(hidden, unit);
        pack_w = hidden % unit != 0 || p.weight.ld % unit != 0 || reinterpret_cast<uintptr_t>(p.weight.data) % 16 != 0;
        const uint64_t row = backward ? tokens * size : pack_w ? padded * size : 1;
        piece = std::min(std::max<uint64_t>(kPieceBytes / std::max<uint64_t>(row, 1) / 256 * 256, 2048), roundUp(classes, 256));
        parts = ceilDiv(classes, headPartClasses(p.type));
        const uint64_t tile  = p.type == FTRAIN_NUMERIC_TYPE_FP32 ? 128 : 256;
        const uint64_t tiles = std::max<uint64_t>(1, ceilDiv(tokens, tile) * ceilDiv(hidden, tile));
        slices               = static_cast<int>(std::max<uint64_t>(1, std::min(kFill / tiles, static_cast<uint64_t>(piece) / 512)));
        slice                = tokens * padded;
        auto take            = [&](uint64_t n) {
            const uint64_t at = bytes;
            bytes += roundUp(n, 256);
            return at;
        };
        head  = take(sizeof(Head));
        place = take(tokens * 4);
        rows  = take(tokens * sizeof(RowInfo));
        x     = take(tokens * padded * size);
        w     = pack_w ? take(piece * padded * size) : 0;
        part  = backward ? 0 : take(tokens * parts * sizeof(float2));
        hit   = backward ? 0 : take(tokens * 4);
        dl    = backward ? take(tokens * piece * size) : 0;
        dx    = backward ? take(slices * slice * 4) : 0;
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

// The classes from `first` on, `n` of them, in rows of whole 16-byte units.
template <class T>
const T* weightPiece(const CrossEntropy& p, const Layout& l, char* base, int64_t first, int64_t n, int64_t& ld,
                     hipStream_t stream) {
    const T* const from = static_cast<const T*>(p.weight.data) + first * p.weight.ld;
    ld                  = p.weight.ld;
    if (!l.pack_w) return from;
    T* const to = reinterpret_cast<T*>(base + l.w);
    launch(&copyRows<T>, "cross entropy weight copy", dim3(static_cast<uint32_t>(std::min<int64_t>(n, 65536))), dim3(kThreads),
           stream, from, p.weight.ld, n, p.weight.cols, to, l.padded, l.padded, static_cast<const int32_t*>(nullptr));
    ld = l.padded;
    return to;
}

template <class T>
void forward(const CrossEntropy& p, char* base, hipStream_t stream) {
    const Layout l(p, false);
    const Buffers b = packInputs<T>(p, l, base, false, stream);
    HeadTileArgs t{};
    t.a = base + l.x, t.lda = l.padded;
    t.m = p.hidden.rows, t.k = l.padded;
    t.head = b.head, t.rows = b.rows;
    t.part = reinterpret_cast<float2*>(base + l.part), t.hit = reinterpret_cast<float*>(base + l.hit);
    t.parts              = l.parts;
    const int64_t classes = p.weight.rows, piece = l.pack_w ? l.piece : classes;
    for (int64_t v = 0; v < classes; v += piece) {
        t.n = std::min(piece, classes - v), t.first_class = v;
        t.b = weightPiece<T>(p, l, base, v, t.n, t.ldb, stream);
        launchHeadTile(p.type, HeadTile::kLogSum, t, 1, stream);
    }
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
    const int64_t unit = 16 / sizeof(T);
    for (int64_t v = 0; v < classes; v += l.piece) {
        HeadTileArgs t{};
        t.head = b.head, t.rows = b.rows, t.first_class = v;
        const int64_t n = std::min(l.piece, classes - v);
        int64_t ldw;
        const T* const w = weightPiece<T>(p, l, base, v, n, ldw, stream);
        if (tokens > 0) {
            t.a = base + l.x, t.lda = l.padded;
            t.b = w, t.ldb = ldw;
            t.d = base + l.dl, t.ldd = l.piece;
            t.m = tokens, t.n = n, t.k = l.padded;
            launchHeadTile(p.type, HeadTile::kGradLogits, t, 1, stream);
            t.a = base + l.dl, t.lda = l.piece;
            t.d = base + l.dx, t.ldd = l.padded;
            t.n = l.padded, t.k = n;
            // Whole stages of the tile to a slice; a last piece's slices may be fewer, its sums then
            // leave the others as they are.
            t.k_chunk        = roundUp(ceilDiv(n, l.slices), 64);
            t.slice          = l.slice;
            t.add            = v > 0;
            const int slices = t.add ? static_cast<int>(ceilDiv(n, t.k_chunk)) : l.slices;
            launchHeadTile(p.type, HeadTile::kGradHidden, t, slices, stream);
        }
        t.a = base + l.dl, t.lda = l.piece;
        t.b = base + l.x, t.ldb = l.padded;
        t.d = static_cast<T*>(p.grad_weight.data) + v * p.grad_weight.ld, t.ldd = p.grad_weight.ld;
        t.m = n, t.n = hidden, t.k = tokens;
        t.read_m = roundUp(n, unit), t.read_n = l.padded;
        launchHeadTile(p.type, HeadTile::kGradWeight, t, 1, stream);
    }
    if (tokens > 0)
        launch(&finishHidden<T>, "cross entropy hidden gradient's rows",
               dim3(static_cast<uint32_t>(std::min<int64_t>(tokens, 65536))), dim3(kThreads), stream,
               reinterpret_cast<const float*>(base + l.dx), l.padded, static_cast<const int32_t*>(b.place),
               static_cast<const Head*>(b.head), static_cast<T*>(p.grad_hidden.data), p.grad_hidden.ld, tokens, hidden,
               l.slices, l.slice);
}

}  // namespace

int headPartClasses(FTrainNumericType type) { return type == FTRAIN_NUMERIC_TYPE_FP32 ? 64 : 256; }

void launchHeadTile(FTrainNumericType type, HeadTile what, const HeadTileArgs& args, int slices, hipStream_t stream) {
    if (type == FTRAIN_NUMERIC_TYPE_FP32)
        launchHeadTileFp32(what, args, slices, stream);
    else if (type == FTRAIN_NUMERIC_TYPE_BF16)
        launchHeadTileBf16(what, args, slices, stream);
    else
        launchHeadTileFp16(what, args, slices, stream);
}

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
