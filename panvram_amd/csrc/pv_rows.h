// What the norms' kernels (pv_norm.hip, pv_layer.hip) share: rows held in registers, sums over a row, and the sum of the partial
// gradients of a row of weights.
#pragma once
#include "pv_ops.h"

namespace pvo {

constexpr int PARTS = 1024;                 // workgroups of the backward pass at most: rows of partial weight gradients

// One row: D elements as packs of P, pack k * LANES + lane in register k of a lane; PACKS 0: not held, any number of packs.
// ROWS: rows at a time of a workgroup
template <int LANES_, int PACKS_, int ROWS_> struct Plan {
    static constexpr int LANES = LANES_, PACKS = PACKS_, ROWS = ROWS_;
    static constexpr int BLOCK = LANES * ROWS, WAVES = LANES > WAVE ? LANES / WAVE : 1;
};

// A sum, or a largest value, over the lanes of a row
template <typename L, typename T, typename F> __device__ inline T over_row(T x, T* lds, F&& join) {
#pragma unroll
    for (int d = (L::LANES < WAVE ? L::LANES : WAVE) / 2; d; d >>= 1) x = join(x, T(__shfl_xor(x, d, WAVE)));
    if constexpr (L::WAVES > 1) {
        const int row = threadIdx.x / L::LANES, wave = threadIdx.x / WAVE;
        __syncthreads();                                       // the last use of lds is over
        if (threadIdx.x % WAVE == 0) lds[wave] = x;
        __syncthreads();
        x = lds[row * L::WAVES];
#pragma unroll
        for (int w = 1; w < L::WAVES; w++) x = join(x, lds[row * L::WAVES + w]);
    }
    return x;
}
template <typename L> __device__ inline float row_sum(float x, float* lds) {
    return over_row<L>(x, lds, [](float a, float b) { return a + b; });
}

// A pack of a row at element i of D: whole, or a part of one at the row's end
template <int P, bool ONCE, typename T> __device__ inline pack<T, P> take(const T* row, int64_t i, int64_t D) {
    if (i + P <= D) return ONCE ? pack<T, P>::load_once(row + i) : pack<T, P>::load(row + i);
    return pack<T, P>::load_part(row + i, D - i);
}
template <bool ONCE, typename T, int P> __device__ inline void leave(const pack<T, P>& v, T* row, int64_t i, int64_t D) {
    if (i + P > D) v.store_part(row + i, D - i);
    else if (ONCE) v.store_once(row + i);
    else v.store(row + i);
}

// d_weight[i] = sum of the partial rows, from column `first` on: 64 columns a workgroup, its 16 waves a run of rows each. The grid's
// second row does the same for d_second, whose partial rows lie behind.
constexpr int END_WAVES = 16;
static __global__ __launch_bounds__(END_WAVES* WAVE) void norm_weight_kernel(const float* __restrict__ parts, int64_t rows, int64_t D, int64_t first, float* __restrict__ d_weight,
                                                                           float* __restrict__ d_second) {
    __shared__ float lds[END_WAVES][WAVE];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const int64_t i = first + int64_t(blockIdx.x) * WAVE + lane;
    float sum = 0.0f;
    parts += blockIdx.y * rows * D;
    if (i < D) {
#pragma unroll 8
        for (int64_t k = wave; k < rows; k += END_WAVES) sum += parts[k * D + i];
    }
    lds[wave][lane] = sum;
    __syncthreads();
    if (wave || i >= D) return;
#pragma unroll
    for (int w = 1; w < END_WAVES; w++) sum += lds[w][lane];
    (blockIdx.y ? d_second : d_weight)[i] = sum;
}

inline int64_t groups_of(int64_t N, int rows) { const int64_t g = (N + rows - 1) / rows; return g < PARTS ? g : PARTS; }

}  // namespace pvo
