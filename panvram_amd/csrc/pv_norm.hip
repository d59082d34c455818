// The residual stream's addition and its root-mean-square norm, in the stream's type or in 8 bits, and the gradients.
//
//   s = x + residual, rounded to the stream's type: what the next layer adds to, and what is normalised
//   r = 1 / sqrt(mean(s^2) + eps),  y = s r weight
//   8 bits: scale = max |y| / the largest value of the format, per row; q = round(y / scale)
//   backward, with u = s r and g = d_y weight:  d = d_stream + r (g - u mean(g u));  d_weight = sum over rows of d_y u
// One wave per row; sums in 32 bits. Every byte is read and written once but for the row that a second pass takes from the
// caches.
#include "pv_ops.h"

using namespace pvo;

namespace {

constexpr int ROWS = 4;                    // waves, and rows at a time, of a workgroup
constexpr int BLOCK = ROWS * WAVE;
constexpr int PARTS = 256;                 // workgroups of the backward pass at most: rows of partial weight gradients

__device__ inline float wave_max_nan(float x) {       // the largest, or NaN if there is one
#pragma unroll
    for (int d = WAVE / 2; d; d >>= 1) {
        const float o = __shfl_xor(x, d, WAVE);
        x = o != o || o > x ? o : x;
    }
    return x;
}

struct Fp8 {
    using type = uint8_t;
    static constexpr float MOST = 448.0f;
    // (|v| is at most 448 but for the quotient's rounding, and what is nearer to 448 than to 480 rounds to it; NaN stays NaN)
    static __device__ type make(float v) { return uint8_t(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false)); }
};
struct Int8 {
    using type = int8_t;
    static constexpr float MOST = 127.0f;
    static __device__ type make(float v) { return v != v ? 0 : int8_t(fminf(fmaxf(rintf(v), -127.0f), 127.0f)); }
};

template <typename E, typename Q>
__global__ __launch_bounds__(BLOCK) void norm_kernel(const E* x, const E* residual, const float* weight, int64_t N, int64_t D, int64_t xs, int64_t rs,
                                                     float eps, E* y, E* stream, float* rstd, typename Q::type* q, float* scale) {
    const int lane = threadIdx.x % WAVE;
    const int64_t n = int64_t(blockIdx.x) * ROWS + threadIdx.x / WAVE;
    if (n >= N) return;
    const E* row = x + n * xs;
    float sum = 0.0f;
    for (int64_t i = lane; i < D; i += WAVE) {
        float s = float(row[i]);
        if (residual) {
            const E t = E(s + float(residual[n * rs + i]));
            stream[n * D + i] = t;
            s = float(t);
        }
        sum = fmaf(s, s, sum);
    }
    const E* from = residual ? stream + n * D : row;
    sum = wave_sum(sum);
    float r = rsqrtf(sum / float(D) + eps);
    if (sum == INFINITY) {                 // squares over 2^128: once more of 2^-64 s
        sum = 0.0f;
        for (int64_t i = lane; i < D; i += WAVE) { const float s = 0x1p-64f * float(from[i]); sum = fmaf(s, s, sum); }
        r = 0x1p-64f * rsqrtf(wave_sum(sum) / float(D) + 0x1p-128f * eps);
    }
    if (rstd && lane == 0) rstd[n] = r;
    if (y) {
        for (int64_t i = lane; i < D; i += WAVE) y[n * D + i] = E(float(from[i]) * r * weight[i]);
        return;
    }
    float most = 0.0f;
    for (int64_t i = lane; i < D; i += WAVE) {
        const float a = fabsf(float(from[i]) * r * weight[i]);
        most = a != a || a > most ? a : most;
    }
    const float sc = wave_max_nan(most) / Q::MOST;
    if (lane == 0) scale[n] = sc;
    for (int64_t i = lane; i < D; i += WAVE) q[n * D + i] = Q::make(sc == 0.0f ? 0.0f : float(from[i]) * r * weight[i] / sc);
}

template <typename E>
__global__ __launch_bounds__(BLOCK) void norm_back_kernel(const E* s, const float* rstd, const float* weight, int64_t N, int64_t D, int64_t ss, const E* d_y,
                                                          const E* d_stream, E* d, float* parts) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    float* part = parts + (int64_t(blockIdx.x) * ROWS + wave) * D;
    for (int64_t i = lane; i < D; i += WAVE) part[i] = 0.0f;
    for (int64_t n = int64_t(blockIdx.x) * ROWS + wave; n < N; n += int64_t(gridDim.x) * ROWS) {
        const float r = rstd[n];
        float sum = 0.0f;
        for (int64_t i = lane; i < D; i += WAVE) {
            const float u = float(s[n * ss + i]) * r, dy = float(d_y[n * D + i]);
            sum = fmaf(dy * weight[i], u, sum);
            part[i] = fmaf(dy, u, part[i]);
        }
        const float m = wave_sum(sum) / float(D);
        for (int64_t i = lane; i < D; i += WAVE) {
            const float u = float(s[n * ss + i]) * r, g = float(d_y[n * D + i]) * weight[i];
            d[n * D + i] = E((d_stream ? float(d_stream[n * D + i]) : 0.0f) + r * (g - u * m));
        }
    }
}

__global__ __launch_bounds__(BLOCK) void norm_weight_kernel(const float* parts, int64_t rows, int64_t D, float* d_weight) {
    const int64_t i = int64_t(blockIdx.x) * BLOCK + threadIdx.x;
    if (i >= D) return;
    float sum = 0.0f;
    for (int64_t k = 0; k < rows; k++) sum += parts[k * D + i];
    d_weight[i] = sum;
}

int64_t parts_of(int64_t N) { const int64_t g = (N + ROWS - 1) / ROWS; return g < PARTS ? g : PARTS; }

int32_t check(int64_t N, int64_t D, int32_t dtype, char* err, size_t cap) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, cap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (N < 0 || D < 1 || N > int64_t(ROWS) * INT32_MAX) return fail(PV_EARG, err, cap, "shape: 0 <= N < 2^33, D >= 1");
    return PV_OK;
}

template <typename Q>
int32_t forward(const void* x, const void* residual, const float* weight, int64_t N, int64_t D, int64_t xs, int64_t rs, float eps, int32_t dtype, void* y,
                void* stream_out, float* rstd, void* q, float* scale, void* stream, char* err, size_t errcap) {
    if (int32_t e = check(N, D, dtype, err, errcap)) return e;
    if (!N) return PV_OK;
    if (!x || !weight || (residual && !stream_out) || (!y && (!q || !scale))) return fail(PV_EARG, err, errcap, "null argument");
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        norm_kernel<E, Q><<<dim3((N + ROWS - 1) / ROWS), BLOCK, 0, hipStream_t(stream)>>>(
            static_cast<const E*>(x), static_cast<const E*>(residual), weight, N, D, xs, rs, eps, static_cast<E*>(y), static_cast<E*>(stream_out), rstd,
            static_cast<typename Q::type*>(q), scale);
        return launched(err, errcap);
    });
}

}  // namespace

extern "C" {

int32_t pv_add_rms_norm_hip(const void* x, const void* residual, const float* weight, int64_t N, int64_t D, int64_t x_row, int64_t residual_row, float eps,
                            int32_t dtype, void* y, void* stream_out, float* rstd, void* stream, char* err, size_t errcap) {
    if (N && !y) return fail(PV_EARG, err, errcap, "null argument");
    return forward<Fp8>(x, residual, weight, N, D, x_row, residual_row, eps, dtype, y, stream_out, rstd, nullptr, nullptr, stream, err, errcap);
}

int32_t pv_add_rms_norm_8bit_hip(const void* x, const void* residual, const float* weight, int64_t N, int64_t D, int64_t x_row, int64_t residual_row, float eps,
                                 int32_t dtype, int32_t format, void* q, float* scale, void* stream_out, void* stream, char* err, size_t errcap) {
    if (format == PV_E4M3)
        return forward<Fp8>(x, residual, weight, N, D, x_row, residual_row, eps, dtype, nullptr, stream_out, nullptr, q, scale, stream, err, errcap);
    if (format == PV_INT8)
        return forward<Int8>(x, residual, weight, N, D, x_row, residual_row, eps, dtype, nullptr, stream_out, nullptr, q, scale, stream, err, errcap);
    return fail(PV_EARG, err, errcap, "format: PV_E4M3 or PV_INT8");
}

uint64_t pv_add_rms_norm_work_bytes(int64_t N, int64_t D) { return N > 0 && D > 0 ? uint64_t(parts_of(N)) * ROWS * uint64_t(D) * 4 : 0; }

int32_t pv_add_rms_norm_backward_hip(const void* s, const float* rstd, const float* weight, int64_t N, int64_t D, int64_t s_row, const void* d_y,
                                     const void* d_stream, int32_t dtype, void* d, float* d_weight, void* work, uint64_t work_bytes, void* stream, char* err,
                                     size_t errcap) {
    if (int32_t e = check(N, D, dtype, err, errcap)) return e;
    if (!d_weight || (N && (!s || !rstd || !weight || !d_y || !d))) return fail(PV_EARG, err, errcap, "null argument");
    if (work_bytes < pv_add_rms_norm_work_bytes(N, D) || (N && !work)) return fail(PV_EARG, err, errcap, "work: too small");
    const hipStream_t st = hipStream_t(stream);
    float* parts = static_cast<float*>(work);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        const int64_t g = parts_of(N);
        if (N) norm_back_kernel<E><<<dim3(g), BLOCK, 0, st>>>(static_cast<const E*>(s), rstd, weight, N, D, s_row, static_cast<const E*>(d_y),
                                                              static_cast<const E*>(d_stream), static_cast<E*>(d), parts);
        norm_weight_kernel<<<dim3((D + BLOCK - 1) / BLOCK), BLOCK, 0, st>>>(parts, g * ROWS, D, d_weight);
        return launched(err, errcap);
    });
}

}  // extern "C"
