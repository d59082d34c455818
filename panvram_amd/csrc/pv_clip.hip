// The norm over many gradient tensors, and the tensors scaled so that it is at most max_norm.
//
//   norm = sqrt(sum over all tensors of the sum of their squares);  factor = min(1, max_norm / (norm + 1e-6))
// Squares are taken and summed in 64 bits: those of large or tiny 32-bit gradients neither overflow nor vanish, and the order
// of the sums is fixed. A NaN or an infinity reaches the norm. One launch takes up to GROUP tensors by value, so that nothing
// has to be copied to the device first and a call may be captured into a graph.
#include "pv_ops.h"

using namespace pvo;

namespace {

constexpr int GROUP = 120;                 // tensors of one launch: 28 bytes each of the 4 KiB that a launch's arguments may take
constexpr int BLOCK = 256;
constexpr int64_t PIECE = 16384;           // elements of a workgroup

struct Group {
    const void* from[GROUP];
    void* to[GROUP];
    int64_t n[GROUP];
    uint32_t first[GROUP];                 // workgroup that begins a tensor
    int32_t count;
};
static_assert(sizeof(Group) <= 3600, "a launch's arguments");

// The tensor that workgroup `b` works on: the last that begins at or before it
__device__ inline int tensor_of(const Group& G, uint32_t b) {
    int lo = 0, hi = G.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (G.first[mid] <= b) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ inline double block_sum(double x) {
    __shared__ double lds[BLOCK / WAVE];
#pragma unroll
    for (int d = WAVE / 2; d; d >>= 1) x += __shfl_xor(x, d, WAVE);
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = x;
    __syncthreads();
    double sum = 0.0;
    for (int w = 0; w < BLOCK / WAVE; w++) sum += lds[w];
    return sum;
}

template <typename E> __global__ __launch_bounds__(BLOCK) void square_kernel(Group G, double* parts) {
    const int k = tensor_of(G, blockIdx.x);
    const E* g = static_cast<const E*>(G.from[k]);
    const int64_t i0 = int64_t(blockIdx.x - G.first[k]) * PIECE, i1 = i0 + PIECE < G.n[k] ? i0 + PIECE : G.n[k];
    double sum = 0.0;
    for (int64_t i = i0 + threadIdx.x; i < i1; i += BLOCK) { const double x = double(float(g[i])); sum = fma(x, x, sum); }
    sum = block_sum(sum);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

__global__ __launch_bounds__(BLOCK) void norm_end_kernel(const double* parts, int64_t n, float* norm) {
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += BLOCK) sum += parts[i];
    sum = block_sum(sum);
    if (threadIdx.x == 0) *norm = float(sqrt(sum));
}

template <typename E> __global__ __launch_bounds__(BLOCK) void scale_kernel(Group G, const float* norm, float max_norm) {
    const float c = max_norm / (*norm + 1e-6f);
    const float factor = c > 1.0f ? 1.0f : c;          // (NaN stays)
    const int k = tensor_of(G, blockIdx.x);
    const E* g = static_cast<const E*>(G.from[k]);
    E* o = static_cast<E*>(G.to[k]);
    if (factor == 1.0f && g == o) return;
    const int64_t i0 = int64_t(blockIdx.x - G.first[k]) * PIECE, i1 = i0 + PIECE < G.n[k] ? i0 + PIECE : G.n[k];
    for (int64_t i = i0 + threadIdx.x; i < i1; i += BLOCK) o[i] = E(float(g[i]) * factor);
}

uint64_t blocks_of(int64_t n) { return uint64_t((n + PIECE - 1) / PIECE); }

// Groups of up to GROUP tensors of one type, in order; f(group, workgroups, workgroups of the type's earlier groups)
template <typename F> void groups(const void* const* from, void* const* to, const int64_t* n, const int32_t* dtypes, int32_t count, int32_t dtype, F&& f) {
    Group G;
    G.count = 0;
    uint64_t blocks = 0;
    for (int32_t i = 0; i < count; i++) {
        if (dtypes[i] != dtype || !n[i]) continue;
        const uint64_t b = blocks_of(n[i]);
        if (G.count == GROUP || (G.count && blocks + b > INT32_MAX)) {
            f(G, uint32_t(blocks));
            G.count = 0;
            blocks = 0;
        }
        G.from[G.count] = from[i];
        G.to[G.count] = to ? to[i] : nullptr;
        G.n[G.count] = n[i];
        G.first[G.count++] = uint32_t(blocks);
        blocks += b;
    }
    if (G.count) f(G, uint32_t(blocks));
}

}  // namespace

extern "C" {

uint64_t pv_gradient_norm_work_bytes(const int64_t* sizes, int32_t count) {
    uint64_t b = 0;
    for (int32_t i = 0; sizes && i < count; i++) if (sizes[i] > 0) b += blocks_of(sizes[i]);
    return b * 8;
}

int32_t pv_gradient_norm_hip(const void* const* grads, void* const* out, const int64_t* sizes, const int32_t* dtypes, int32_t count, float max_norm, float* norm,
                             void* work, uint64_t work_bytes, void* stream, char* err, size_t errcap) {
    if (count < 0 || !norm || (count && (!grads || !sizes || !dtypes))) return fail(PV_EARG, err, errcap, "null argument");
    for (int32_t i = 0; i < count; i++) {
        if (!element_bytes(dtypes[i])) return fail(PV_EARG, err, errcap, "dtype: one of PV_F32, PV_BF16, PV_F16");
        if (sizes[i] < 0 || blocks_of(sizes[i]) > INT32_MAX) return fail(PV_EARG, err, errcap, "size: 0 to 2^45 elements");
        if (sizes[i] && (!grads[i] || (out && !out[i]))) return fail(PV_EARG, err, errcap, "null argument");
    }
    const uint64_t need = pv_gradient_norm_work_bytes(sizes, count);
    if (need && (!work || work_bytes < need)) return fail(PV_EARG, err, errcap, "work: too small");
    const hipStream_t st = hipStream_t(stream);
    double* parts = static_cast<double*>(work);
    uint64_t done = 0;
    for (int32_t dtype : {PV_F32, PV_BF16, PV_F16})
        with_type(dtype, [&](auto e) {
            groups(grads, nullptr, sizes, dtypes, count, dtype, [&](const Group& G, uint32_t blocks) {
                square_kernel<decltype(e)><<<blocks, BLOCK, 0, st>>>(G, parts + done);
                done += blocks;
            });
            return 0;
        });
    norm_end_kernel<<<1, BLOCK, 0, st>>>(parts, int64_t(done), norm);
    if (out)
        for (int32_t dtype : {PV_F32, PV_BF16, PV_F16})
            with_type(dtype, [&](auto e) {
                groups(grads, out, sizes, dtypes, count, dtype,
                       [&](const Group& G, uint32_t blocks) { scale_kernel<decltype(e)><<<blocks, BLOCK, 0, st>>>(G, norm, max_norm); });
                return 0;
            });
    return launched(err, errcap);
}

}  // extern "C"
