// The norm over many gradient tensors, and the tensors scaled so that it is at most max_norm.
//
//   norm = sqrt(sum over all tensors of the sum of their squares);  factor = min(1, max_norm / (norm + 1e-6))
// Squares are taken and summed in 64 bits: those of large or tiny 32-bit gradients neither overflow nor vanish, and the order
// of the sums is fixed. A NaN or an infinity reaches the norm. One launch takes up to GROUP tensors by value, so that nothing
// has to be copied to the device first and a call may be captured into a graph.
//
// What bounds it: the bytes, read once for the norm and once more for the scaling where they are more than the caches hold.
// Measured: 500 M bfloat16 elements in 300 tensors, squares 166 us (1.0 GB: 6.0 TB/s), scaling 328 us (2.0 GB: 6.1 TB/s; the last
// tensors first, which the caches may still have). 2 M float32 elements in 150 tensors 17 us in three launches, where the host
// needs 95 us for their addresses, sizes, types and versions.
#include "pv_ops.h"

using namespace pvo;

namespace {

constexpr int GROUP = 160;                 // tensors of one launch: 25 bytes each of the 4 KiB that a launch's arguments may take
constexpr int BLOCK = 256;
// Bytes of a workgroup. Scaling: four loads of 16 bytes a lane (1 GiB read and written in 334 us; 370 with 64 KiB, 394 with 256).
// The sum of squares: the same, or more, so that there are no more than MOST partial sums for one workgroup to add up (1 GiB
// read in 154-166 us with any from 16 to 256 KiB).
constexpr int64_t LINE = BLOCK * 16, PIECE = 4 * LINE, MOST = 4096;

struct Group {
    const void* from[GROUP];
    void* to[GROUP];
    uint32_t first[GROUP];                 // workgroup that begins a tensor
    uint32_t low[GROUP];                   // its elements: low 32 bits, and 6 above them beside the type's 2
    uint8_t high[GROUP];
    int32_t count;
    int64_t piece;                         // bytes of a workgroup
    __host__ __device__ int64_t size(int k) const { return int64_t(high[k] >> 2) << 32 | low[k]; }
    __host__ __device__ int32_t dtype(int k) const { return high[k] & 3; }
};
static_assert(sizeof(Group) <= 4064, "a launch's arguments");
// Workgroups of a launch, and bytes of a tensor, so that its pieces are one launch
constexpr int64_t MOST_BLOCKS = MOST_ITEMS / BLOCK - 1, MOST_BYTES = MOST_BLOCKS * PIECE;

// The tensor that workgroup `b` works on: the last that begins at or before it
__device__ inline int tensor_of(const Group& G, uint32_t b) {
    int lo = 0, hi = G.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (G.first[mid] <= b) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int WAVES> __device__ inline double block_sum(double x) {
    __shared__ double lds[WAVES];
#pragma unroll
    for (int d = WAVE / 2; d; d >>= 1) x += __shfl_xor(x, d, WAVE);
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = x;
    __syncthreads();
    double sum = 0.0;
    for (int w = 0; w < WAVES; w++) sum += lds[w];
    return sum;
}

// A workgroup's part of a tensor of type E: packs of 16 bytes from the first address that is a multiple of 16, and single
// elements before (workgroup 0) and behind them (the last). f(i) and wide(i): element i, and the pack that begins there.
template <typename E, typename F, typename G> __device__ inline void over_part(const E* p, int64_t n, int64_t part, int64_t piece, F&& f, G&& wide) {
    constexpr int P = 16 / sizeof(E);
    int64_t head = (-reinterpret_cast<uintptr_t>(p) & 15) / sizeof(E);
    if (head > n) head = n;
    const int64_t packs = (n - head) / P, per = piece / 16, i0 = part * per, i1 = i0 + per < packs ? i0 + per : packs;
    int64_t i = i0 + threadIdx.x;
    for (; i + 3 * BLOCK < i1; i += 4 * BLOCK) wide(std::integral_constant<int, 4>{}, head + i * P);
    for (; i < i1; i += BLOCK) wide(std::integral_constant<int, 1>{}, head + i * P);
    if (part == 0 && threadIdx.x < head) f(int64_t(threadIdx.x));
    const int64_t tail = head + packs * P;
    if (i0 + per >= packs && i0 <= packs && tail + threadIdx.x < n && (i0 < packs || part == 0)) f(tail + threadIdx.x);
}

__global__ __launch_bounds__(BLOCK) void square_kernel(Group G, double* parts) {
    const int k = tensor_of(G, blockIdx.x);
    double sum[4] = {};
    auto go = [&](auto e) {
        using E = decltype(e);
        const E* g = static_cast<const E*>(G.from[k]);
        constexpr int P = 16 / sizeof(E);
        over_part(g, G.size(k), blockIdx.x - G.first[k], G.piece,
                  [&](int64_t i) { const double x = double(float(g[i])); sum[0] = fma(x, x, sum[0]); },
                  [&](auto many, int64_t i) {
                      constexpr int M = decltype(many)::value;
                      pack<E, P> v[M];
#pragma unroll
                      for (int m = 0; m < M; m++) v[m] = pack<E, P>::load_once(g + i + int64_t(m) * BLOCK * P);
#pragma unroll
                      for (int m = 0; m < M; m++)
#pragma unroll
                          for (int j = 0; j < P; j++) { const double x = double(float(v[m].v[j])); sum[j % 4] = fma(x, x, sum[j % 4]); }
                  });
    };
    if (G.dtype(k) == PV_F32) go(float{}); else if (G.dtype(k) == PV_BF16) go(bf16{}); else go(f16{});
    const double all = block_sum<BLOCK / WAVE>((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (threadIdx.x == 0) parts[blockIdx.x] = all;
}

constexpr int END = 1024;
__global__ __launch_bounds__(END) void norm_end_kernel(const double* parts, int64_t n, float* norm) {
    double sum = 0.0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < n; i += END) sum += parts[i];
    sum = block_sum<END / WAVE>(sum);
    if (threadIdx.x == 0) *norm = float(sqrt(sum));
}

// Last workgroups first: what square_kernel read last may still be in the caches
__global__ __launch_bounds__(BLOCK) void scale_kernel(Group G, const float* norm, float max_norm) {
    const float c = max_norm / (*norm + 1e-6f);
    const float factor = c > 1.0f ? 1.0f : c;          // (NaN stays)
    const uint32_t b = gridDim.x - 1 - blockIdx.x;
    const int k = tensor_of(G, b);
    if (factor == 1.0f && G.from[k] == G.to[k]) return;
    auto go = [&](auto e) {
        using E = decltype(e);
        const E* g = static_cast<const E*>(G.from[k]);
        E* o = static_cast<E*>(G.to[k]);
        constexpr int P = 16 / sizeof(E);
        auto one = [&](int64_t i) { o[i] = E(float(g[i]) * factor); };
        // (o may be off the 16 bytes that g's packs start at)
        over_part(g, G.size(k), b - G.first[k], G.piece, one, [&](auto many, int64_t i) {
            constexpr int M = decltype(many)::value;
            pack<E, P> v[M];
#pragma unroll
            for (int m = 0; m < M; m++) v[m] = pack<E, P>::load_once(g + i + int64_t(m) * BLOCK * P);
#pragma unroll
            for (int m = 0; m < M; m++) {
#pragma unroll
                for (int j = 0; j < P; j++) v[m].v[j] = E(float(v[m].v[j]) * factor);
                v[m].store_once(o + i + int64_t(m) * BLOCK * P);
            }
        });
    };
    if (G.dtype(k) == PV_F32) go(float{}); else if (G.dtype(k) == PV_BF16) go(bf16{}); else go(f16{});
}

int64_t piece_of(const int64_t* sizes, const int32_t* dtypes, int32_t count) {
    int64_t bytes = 0;
    for (int32_t i = 0; i < count; i++) if (sizes[i] > 0) bytes += sizes[i] * element_bytes(dtypes[i]);
    const int64_t piece = (bytes / MOST + LINE - 1) / LINE * LINE;
    return piece > PIECE ? piece : PIECE;
}
int64_t blocks_of(int64_t n, int32_t dtype, int64_t piece) { return (n * element_bytes(dtype) + piece - 1) / piece; }

// f(group, its workgroups) for groups of up to GROUP tensors; `back`: the last first
template <typename F> void groups(const void* const* from, void* const* to, const int64_t* n, const int32_t* dtypes, int32_t count, int64_t piece, bool back, F&& f) {
    Group G;
    G.count = 0;
    G.piece = piece;
    int64_t blocks = 0;
    for (int32_t k = 0; k < count; k++) {
        const int32_t i = back ? count - 1 - k : k;
        if (!n[i]) continue;
        const int64_t more = blocks_of(n[i], dtypes[i], piece);
        if (G.count == GROUP || blocks + more > MOST_BLOCKS) {
            f(G, uint32_t(blocks));
            G.count = 0;
            blocks = 0;
        }
        G.from[G.count] = from[i];
        G.to[G.count] = to ? to[i] : nullptr;
        G.low[G.count] = uint32_t(n[i]);
        G.high[G.count] = uint8_t(n[i] >> 32 << 2 | dtypes[i]);
        G.first[G.count++] = uint32_t(blocks);
        blocks += more;
    }
    if (G.count) f(G, uint32_t(blocks));
}

// What both entries ask of their arguments
int32_t check(const void* const* grads, void* const* out, const int64_t* sizes, const int32_t* dtypes, int32_t count, char* err, size_t cap) {
    if (count < 0 || (count && (!grads || !sizes || !dtypes))) return fail(PV_EARG, err, cap, "null argument");
    int64_t all = 0;
    for (int32_t i = 0; i < count; i++) {
        const int bytes = element_bytes(dtypes[i]);
        if (!bytes) return fail(PV_EARG, err, cap, "dtype: one of PV_F32, PV_BF16, PV_F16");
        if (sizes[i] < 0 || sizes[i] > MOST_BYTES || sizes[i] * bytes > MOST_BYTES || (all += sizes[i]) > (int64_t(1) << 40))
            return fail(PV_EARG, err, cap, "size: 0 elements to less than 2^38 bytes, 2^40 elements in all");
        if (sizes[i] && (!grads[i] || (out && !out[i]))) return fail(PV_EARG, err, cap, "null argument");
        if (sizes[i] && (!aligned(grads[i], bytes) || (out && !aligned(out[i], bytes)))) return fail(PV_EARG, err, cap, "address: not a multiple of the element's size");
    }
    return PV_OK;
}

}  // namespace

extern "C" {

uint64_t pv_gradient_norm_work_bytes(const int64_t* sizes, const int32_t* dtypes, int32_t count) {
    if (!sizes || !dtypes) return 0;
    const int64_t piece = piece_of(sizes, dtypes, count);
    uint64_t b = 0;
    for (int32_t i = 0; i < count; i++) if (sizes[i] > 0) b += uint64_t(blocks_of(sizes[i], dtypes[i], piece));
    return b * 8;
}

int32_t pv_gradient_norm_hip(const void* const* grads, const int64_t* sizes, const int32_t* dtypes, int32_t count, float* norm, void* work, uint64_t work_bytes,
                             void* stream, char* err, size_t errcap) {
    if (!norm) return fail(PV_EARG, err, errcap, "null argument");
    if (int32_t e = check(grads, nullptr, sizes, dtypes, count, err, errcap)) return e;
    const uint64_t need = pv_gradient_norm_work_bytes(sizes, dtypes, count);
    if (need && (!work || work_bytes < need || !aligned(work, 16))) return fail(PV_EARG, err, errcap, "work: too small, or not 16-byte aligned");
    const hipStream_t st = hipStream_t(stream);
    double* parts = static_cast<double*>(work);
    int64_t done = 0;
    groups(grads, nullptr, sizes, dtypes, count, piece_of(sizes, dtypes, count), false, [&](const Group& G, uint32_t blocks) {
        square_kernel<<<blocks, BLOCK, 0, st>>>(G, parts + done);
        done += blocks;
    });
    norm_end_kernel<<<1, END, 0, st>>>(parts, done, norm);
    return launched(err, errcap);
}

int32_t pv_scale_gradients_hip(const void* const* grads, void* const* out, const int64_t* sizes, const int32_t* dtypes, int32_t count, float max_norm,
                               const float* norm, void* stream, char* err, size_t errcap) {
    if (!norm || (count && !out)) return fail(PV_EARG, err, errcap, "null argument");
    if (int32_t e = check(grads, out, sizes, dtypes, count, err, errcap)) return e;
    groups(grads, out, sizes, dtypes, count, PIECE, true,
           [&](const Group& G, uint32_t blocks) { scale_kernel<<<blocks, BLOCK, 0, hipStream_t(stream)>>>(G, norm, max_norm); });
    return launched(err, errcap);
}

}  // extern "C"
