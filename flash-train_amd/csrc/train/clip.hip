// The global norm of many gradients, and clipping:
//   norm = sqrt(sum over all tensors of g^2),  out = g min(1, max_norm / (norm + eps)).
//
// Two launches for every kBatch tensors: `sumSquares` leaves one partial sum per workgroup, `scale`
// adds the partials up (every workgroup for itself, in one order) and writes the outputs.  The
// tensors' addresses travel in the kernel arguments: nothing is copied to the device, so a captured
// graph holds them.  Squares and sums are in 64 bits: the square of a large fp32 or bf16 gradient
// overflows 32 bits.
#include "device.hpp"
#include "ft/train.hpp"

namespace ftrain::train {
namespace {

constexpr int kThreads = 256;
// Workgroups: eight of 256 threads on each of the 256 CUs.
constexpr int kGrid = 2048;
// Elements a workgroup takes at a time.
constexpr uint64_t kChunk = 16384;
// Tensors of one launch: their descriptions fill most of the 4 KiB that kernel arguments may take.
constexpr int kBatch = 112;

struct Batch {
    const void* in[kBatch];
    void* out[kBatch];
    uint64_t count[kBatch];
    uint32_t first[kBatch];  // each tensor's first chunk
    uint8_t type[kBatch];
    uint32_t chunks;
    int32_t n;
};

template <class T, class F>
__device__ __forceinline__ void eachPack(const T* in, uint64_t begin, uint64_t end, F&& f) {
    constexpr int N = Pack<T>::kCount;
    const uint64_t whole = begin + (end - begin) / N * N;
#pragma unroll 4
    for (uint64_t i = begin + threadIdx.x * N; i < whole; i += kThreads * N)
        f(i, *reinterpret_cast<const Pack<T>*>(in + i), N);
    if (whole + threadIdx.x < end) {
        Pack<T> one{};
        one.v[0] = in[whole + threadIdx.x];
        f(whole + threadIdx.x, one, 1);
    }
}

// f(tensor, first element, past the last element) for the workgroup's chunks of the batch, from the
// first to the last or back.  The lanes hold the tensors' first chunks, and a chunk's tensor is the last
// that starts no later: kernel arguments are in host memory, where each step of a search of them waits
// about a microsecond.
template <class F>
__device__ __forceinline__ void eachChunk(const Batch& b, bool back, F&& f) {
    static_assert(kBatch <= 2 * kWave, "two tensors a lane");
    const int lane      = threadIdx.x % kWave;
    const uint32_t low  = lane < b.n ? b.first[lane] : UINT32_MAX;
    const uint32_t high = lane + kWave < b.n ? b.first[lane + kWave] : UINT32_MAX;
    for (uint32_t c = blockIdx.x; c < b.chunks; c += gridDim.x) {
        const uint32_t chunk = back ? b.chunks - 1 - c : c;
        const int t          = __popcll(__ballot(low <= chunk)) + __popcll(__ballot(high <= chunk)) - 1;
        const uint64_t begin = static_cast<uint64_t>(chunk - b.first[t]) * kChunk;
        f(t, begin, min(begin + kChunk, b.count[t]));
    }
}

__device__ __forceinline__ double blockSum(double v) {
    __shared__ double part[kThreads / kWave];
    v = groupSum<kWave>(v);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kThreads / kWave; ++i) v += part[i];
    return v;
}

__global__ __launch_bounds__(kThreads) void sumSquares(Batch b, double* partials, bool add) {
    double sum = 0.0;
    auto run = [&](auto* in, uint64_t begin, uint64_t end) {
        eachPack(in, begin, end, [&](uint64_t, const auto& p, int n) {
#pragma unroll
            for (int e = 0; e < p.kCount; ++e) {
                const double x = toFloat(p.v[e]);
                if (e < n) sum = fma(x, x, sum);
            }
        });
    };
    eachChunk(b, false, [&](int t, uint64_t begin, uint64_t end) {
        if (b.type[t] == FTRAIN_NUMERIC_TYPE_FP32)
            run(static_cast<const float*>(b.in[t]), begin, end);
        else if (b.type[t] == FTRAIN_NUMERIC_TYPE_BF16)
            run(static_cast<const bf16*>(b.in[t]), begin, end);
        else
            run(static_cast<const fp16*>(b.in[t]), begin, end);
    });
    sum = blockSum(sum);
    if (threadIdx.x == 0) partials[blockIdx.x] = add ? partials[blockIdx.x] + sum : sum;
}

__global__ __launch_bounds__(kThreads) void scale(Batch b, const double* partials, int n, float max_norm, float eps,
                                                  float* norm_out) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) sum += partials[i];
    const float norm = static_cast<float>(sqrt(blockSum(sum)));
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    float coef = max_norm / (norm + eps);
    if (coef > 1.f) coef = 1.f;  // a NaN stays
    auto run = [&](auto* in, auto* out, uint64_t begin, uint64_t end) {
        using T = std::remove_pointer_t<decltype(out)>;
        eachPack(in, begin, end, [&](uint64_t i, const auto& p, int count) {
            Pack<T> r;
#pragma unroll
            for (int e = 0; e < p.kCount; ++e) r.v[e] = static_cast<T>(toFloat(p.v[e]) * coef);
            if (count == p.kCount)
                *reinterpret_cast<Pack<T>*>(out + i) = r;
            else
                out[i] = r.v[0];
        });
    };
    eachChunk(b, true, [&](int t, uint64_t begin, uint64_t end) {
        if (coef == 1.f && b.in[t] == b.out[t]) return;
        if (b.type[t] == FTRAIN_NUMERIC_TYPE_FP32)
            run(static_cast<const float*>(b.in[t]), static_cast<float*>(b.out[t]), begin, end);
        else if (b.type[t] == FTRAIN_NUMERIC_TYPE_BF16)
            run(static_cast<const bf16*>(b.in[t]), static_cast<bf16*>(b.out[t]), begin, end);
        else
            run(static_cast<const fp16*>(b.in[t]), static_cast<fp16*>(b.out[t]), begin, end);
    });
}

// f(batch) for the tensors in order; empty ones are left out.  At least one call.
template <class F>
void eachBatch(const ClipTensor* tensors, std::size_t n, F&& f) {
    Batch b{};
    bool any = false;
    for (std::size_t i = 0; i < n; ++i) {
        const ClipTensor& t = tensors[i];
        if (t.count == 0) continue;
        const uint64_t chunks = (t.count + kChunk - 1) / kChunk;
        if (b.n == kBatch || (b.n > 0 && b.chunks + chunks > UINT32_MAX / 2)) {
            f(b);
            any = true;
            b   = Batch{};
        }
        b.in[b.n]    = t.in;
        b.out[b.n]   = t.out;
        b.count[b.n] = t.count;
        b.first[b.n] = b.chunks;
        b.type[b.n]  = t.type;
        b.chunks += static_cast<uint32_t>(chunks);
        ++b.n;
    }
    if (b.n > 0 || !any) f(b);
}

}  // namespace

uint64_t clipWorkspace() { return kGrid * sizeof(double); }

void clipGradNorm(const ClipTensor* tensors, std::size_t n, float* norm, float max_norm, float eps, void* workspace,
                  hipStream_t stream) {
    uint32_t grid = 1;
    eachBatch(tensors, n, [&](const Batch& b) { grid = std::max(grid, std::min<uint32_t>(b.chunks, kGrid)); });
    auto* partials = static_cast<double*>(workspace);
    bool add       = false;
    eachBatch(tensors, n, [&](const Batch& b) {
        launch(sumSquares, "clip sum", dim3(grid), dim3(kThreads), stream, b, partials, add);
        add = true;
    });
    float* out = norm;
    eachBatch(tensors, n, [&](const Batch& b) {
        launch(scale, "clip scale", dim3(grid), dim3(kThreads), stream, b, static_cast<const double*>(partials),
               static_cast<int>(grid), max_norm, eps, out);
        out = nullptr;
    });
}

}  // namespace ftrain::train
