// The head and loss of a model that predicts the next token of a window over a small alphabet, and the gradients.
//
//   logits[b, t, v] = hidden[b, t, :] . weight[v, :];  a place (b, t) counts if tokens[b, t + 1] is one of the V ids and not
//   `ignore` (the last place of a row never does);  each = logsumexp(logits) - logits[tokens[b, t + 1]], 0 where nothing
//   counts;  loss = sum of each / number of places that count (0 where there are none)
//   d_logits = (softmax - onehot) * w, w = scale / count or the place's own factor;
//   d_hidden = d_logits weight (0 where a place does not count);  d_weight = sum over places of d_logits^T hidden
// What stands in hidden at places that do not count (NaN too) reaches nothing.
#include "pv_ops.h"

using namespace pvo;

namespace {

constexpr int VMAX = 16;                   // ids at most
constexpr int ROWS = 4;                    // waves, and places at a time, of a workgroup
constexpr int BLOCK = ROWS * WAVE;
constexpr int COUNTS = 256;                // workgroups that count places
constexpr int SPLITS = 64;                 // runs of places in which weight gradients are summed

struct Shape {
    int64_t B, T, D, hb, ht, tb;           // strides in elements: hidden (batch, time), tokens (batch); channels, tokens are neighbours
    int64_t ignore;
    int32_t V;
};

// the id that place n predicts, or -1 where it does not count
template <typename I> __device__ inline int target(const Shape& S, const I* tokens, int64_t n) {
    const int64_t b = n / S.T, t = n % S.T;
    if (t + 1 >= S.T) return -1;
    const int64_t v = int64_t(tokens[b * S.tb + t + 1]);
    return v >= 0 && v < S.V && v != S.ignore ? int(v) : -1;
}

template <typename X> __device__ inline X block_sum(X x, X* lds) {
#pragma unroll
    for (int d = WAVE / 2; d; d >>= 1) x += __shfl_xor(x, d, WAVE);
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = x;
    __syncthreads();
    X sum = 0;
    for (int w = 0; w < int(blockDim.x) / WAVE; w++) sum += lds[w];
    __syncthreads();
    return sum;
}

template <typename I> __global__ __launch_bounds__(BLOCK) void loss_count_kernel(Shape S, const I* tokens, int64_t* counts) {
    __shared__ int64_t lds[ROWS];
    int64_t k = 0;
    for (int64_t n = int64_t(blockIdx.x) * BLOCK + threadIdx.x; n < S.B * S.T; n += int64_t(gridDim.x) * BLOCK) k += target(S, tokens, n) >= 0;
    k = block_sum(k, lds);
    if (threadIdx.x == 0) counts[blockIdx.x] = k;
}

template <typename E, typename W, typename I>
__global__ __launch_bounds__(BLOCK) void loss_place_kernel(Shape S, const E* hidden, const W* weight, const I* tokens, const int64_t* counts, const float* scale,
                                                           const float* factor, float* each, E* d_hidden, float* d_logits, double* sums) {
    __shared__ int64_t ilds[ROWS];
    __shared__ double dlds[ROWS];
    float base = 1.0f;
    if (counts) {
        const int64_t k = block_sum(counts[threadIdx.x], ilds);
        base = (scale ? *scale : 1.0f) / float(k > 0 ? k : 1);
    }
    const int lane = threadIdx.x % WAVE;
    double sum = 0.0;
    for (int64_t n = int64_t(blockIdx.x) * ROWS + threadIdx.x / WAVE; n < S.B * S.T; n += int64_t(gridDim.x) * ROWS) {
        const int at = target(S, tokens, n);
        const E* h = hidden + n / S.T * S.hb + n % S.T * S.ht;
        float p[VMAX] = {};
        if (at >= 0) {
            for (int64_t i = lane; i < S.D; i += WAVE) {
                const float x = float(h[i]);
#pragma unroll
                for (int v = 0; v < VMAX; v++) if (v < S.V) p[v] = fmaf(x, float(weight[v * S.D + i]), p[v]);
            }
            float top = -INFINITY, total = 0.0f, own = 0.0f;
#pragma unroll
            for (int v = 0; v < VMAX; v++) if (v < S.V) {
                p[v] = wave_sum(p[v]);
                top = fmaxf(top, p[v]);
                if (v == at) own = p[v];
            }
#pragma unroll
            for (int v = 0; v < VMAX; v++) if (v < S.V) { p[v] = expf(p[v] - top); total += p[v]; }
            const float l = logf(total) + top - own;
            if (lane == 0) { if (each) each[n] = l; sum += double(l); }
            if (d_hidden) {
                const float w = factor ? factor[n] : base;
#pragma unroll
                for (int v = 0; v < VMAX; v++) if (v < S.V) p[v] = (p[v] / total - float(v == at)) * w;
            }
        } else if (each && lane == 0) each[n] = 0.0f;
        if (!d_hidden) continue;
        if (lane == 0) for (int v = 0; v < VMAX; v++) d_logits[n * VMAX + v] = v < S.V ? p[v] : 0.0f;
        for (int64_t i = lane; i < S.D; i += WAVE) {
            float x = 0.0f;
#pragma unroll
            for (int v = 0; v < VMAX; v++) if (v < S.V) x = fmaf(p[v], float(weight[v * S.D + i]), x);
            d_hidden[n * S.D + i] = at >= 0 ? E(x) : E(0.0f);
        }
    }
    sum = block_sum(sum, dlds);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// parts[s, v, i]: the sum of one run of places
template <typename E, typename I>
__global__ __launch_bounds__(WAVE) void loss_weight_kernel(Shape S, const E* hidden, const I* tokens, const float* d_logits, float* parts) {
    const int64_t i = int64_t(blockIdx.x) * WAVE + threadIdx.x, N = S.B * S.T, run = (N + SPLITS - 1) / SPLITS;
    const int64_t from = blockIdx.y * run, to = from + run < N ? from + run : N;
    float p[VMAX] = {};
    for (int64_t n = from; n < to; n++) {
        if (target(S, tokens, n) < 0 || i >= S.D) continue;
        const float x = float(hidden[n / S.T * S.hb + n % S.T * S.ht + i]);
#pragma unroll
        for (int v = 0; v < VMAX; v++) p[v] = fmaf(d_logits[n * VMAX + v], x, p[v]);
    }
    if (i >= S.D) return;
    for (int v = 0; v < S.V; v++) parts[(blockIdx.y * int64_t(S.V) + v) * S.D + i] = p[v];
}

template <typename W>
__global__ __launch_bounds__(BLOCK) void loss_end_kernel(Shape S, const int64_t* counts, const double* sums, int nsums, float* loss, const float* parts, W* d_weight) {
    if (blockIdx.x == 0 && loss) {
        __shared__ int64_t ilds[ROWS];
        __shared__ double dlds[ROWS];
        const int64_t k = block_sum(counts[threadIdx.x], ilds);
        double s = 0.0;
        for (int j = threadIdx.x; j < nsums; j += BLOCK) s += sums[j];
        s = block_sum(s, dlds);
        if (threadIdx.x == 0) *loss = float(s / double(k > 0 ? k : 1));
    }
    const int64_t i = int64_t(blockIdx.x) * BLOCK + threadIdx.x;
    if (!d_weight || i >= S.V * S.D) return;
    float x = 0.0f;
    for (int j = 0; j < SPLITS; j++) x += parts[j * int64_t(S.V) * S.D + i];
    d_weight[i] = W(x);
}

constexpr int GRID = 2048;                 // workgroups of loss_place_kernel at most

struct Work { int64_t* counts; double* sums; float* d_logits; float* parts; };
Work layout(void* work, int64_t N) {
    Work w;
    w.counts = static_cast<int64_t*>(work);
    w.sums = reinterpret_cast<double*>(w.counts + COUNTS);
    w.d_logits = reinterpret_cast<float*>(w.sums + GRID);
    w.parts = w.d_logits + N * VMAX;
    return w;
}

template <typename E, typename W, typename I>
int32_t run(const Shape& S, const void* hidden, const void* weight, const void* tokens, const float* scale, const float* factor, float* each, float* loss,
            void* d_hidden, void* d_weight, void* work, hipStream_t st, char* err, size_t errcap) {
    const int64_t N = S.B * S.T;
    const Work w = layout(work, N);
    const int64_t need = (N + ROWS - 1) / ROWS;
    const int grid = int(need < GRID ? need : GRID);
    const I* tok = static_cast<const I*>(tokens);
    const bool mean = loss || !factor;
    static_assert(COUNTS == BLOCK, "one count a lane");
    if (mean) loss_count_kernel<I><<<COUNTS, BLOCK, 0, st>>>(S, tok, w.counts);
    loss_place_kernel<E, W, I><<<grid, BLOCK, 0, st>>>(S, static_cast<const E*>(hidden), static_cast<const W*>(weight), tok, mean ? w.counts : nullptr, scale,
                                                       factor, each, static_cast<E*>(d_hidden), w.d_logits, w.sums);
    if (d_weight)
        loss_weight_kernel<E, I><<<dim3((S.D + WAVE - 1) / WAVE, SPLITS), WAVE, 0, st>>>(S, static_cast<const E*>(hidden), tok, w.d_logits, w.parts);
    if (loss || d_weight)
        loss_end_kernel<W><<<dim3(d_weight ? (S.V * S.D + BLOCK - 1) / BLOCK : 1), BLOCK, 0, st>>>(S, w.counts, w.sums, grid, loss, w.parts, static_cast<W*>(d_weight));
    return launched(err, errcap);
}

}  // namespace

extern "C" {

uint64_t pv_next_base_loss_work_bytes(int64_t B, int64_t T, int64_t D, int32_t V, int32_t gradients) {
    if (B <= 0 || T <= 0 || D <= 0 || V <= 0) return 0;
    const uint64_t head = (COUNTS + GRID) * 8;
    return gradients ? head + uint64_t(B) * T * VMAX * 4 + uint64_t(SPLITS) * V * D * 4 : head;
}

int32_t pv_next_base_loss_hip(const void* hidden, const void* weight, const void* tokens, int64_t B, int64_t T, int64_t D, int32_t V, int64_t hidden_b,
                              int64_t hidden_t, int64_t tokens_b, int64_t ignore, int32_t dtype, int32_t weight_dtype, int32_t token_bytes, const float* scale,
                              const float* factor, float* each, float* loss, void* d_hidden, void* d_weight, void* work, uint64_t work_bytes, void* stream,
                              char* err, size_t errcap) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, errcap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (weight_dtype != dtype && weight_dtype != PV_F32) return fail(PV_EARG, err, errcap, "weight_dtype: hidden's, or PV_F32");
    if (token_bytes != 1 && token_bytes != 8) return fail(PV_EARG, err, errcap, "token_bytes: 1 or 8");
    if (B < 1 || T < 1 || D < 1 || B > (int64_t(1) << 40) / T) return fail(PV_EARG, err, errcap, "shape: B, T, D >= 1, B * T <= 2^40");
    if (V < 1 || V > VMAX) return fail(PV_EARG, err, errcap, "V: 1 to 16 ids");
    if (!hidden || !weight || !tokens || !d_hidden != !d_weight) return fail(PV_EARG, err, errcap, "null argument");
    if (!work || work_bytes < pv_next_base_loss_work_bytes(B, T, D, V, d_hidden != nullptr)) return fail(PV_EARG, err, errcap, "work: too small");
    const Shape S{B, T, D, hidden_b, hidden_t, tokens_b, ignore, V};
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        auto go = [&](auto w) {
            using W = decltype(w);
            if (token_bytes == 1)
                return run<E, W, uint8_t>(S, hidden, weight, tokens, scale, factor, each, loss, d_hidden, d_weight, work, hipStream_t(stream), err, errcap);
            return run<E, W, int64_t>(S, hidden, weight, tokens, scale, factor, each, loss, d_hidden, d_weight, work, hipStream_t(stream), err, errcap);
        };
        return weight_dtype == PV_F32 ? go(float{}) : go(E{});
    });
}

}  // extern "C"
