// The residual stream's addition and its root-mean-square norm, in the stream's type or in 8 bits, and the gradients.
//
//   s = x + residual, rounded to the stream's type: what the next layer adds to, and what is normalised
//   r = 1 / sqrt(mean(s^2) + eps),  y = s r weight
//   8 bits: scale = max |y| / the largest value of the format, per row; q = round(y / scale)
//   backward, with u = s r and g = d_y weight:  d = d_stream + r (g - u mean(g u));  d_weight = sum over rows of d_y u
//
// A row's elements stay in registers between its sums and its outputs: every byte is read once and written once. A row is held
// by LANES lanes, of a wave or of a workgroup, as PACKS packs of 16 bytes a lane (`Plan`); longer rows are read again for each
// pass, from the caches. Rows may begin at any element; a row's last pack may be a part of one. Sums in 32 bits.
//
// What bounds it: the bytes. x, residual, y and all of the backward pass's tensors are passed by the caches, so that the stream,
// which the next layer and the backward pass read, stays in them (65,536 x 1,024 bfloat16 forwards 85 us with this, 98 without,
// backwards 95 and 106; 13,826 x 4,839 float32 171 and 198, 218 and 227. It costs a little where a tensor is no larger than the
// caches or rows are off the lines: 3,487 x 4,127 float32, 58 MB a tensor, 43.5 and 42 us forwards; 65,536 x 513 bfloat16 63 and 57,
// 84 and 80). Measured: 65,536 x 1,024 forwards 80-84 us (537 MB: 6.4-6.7 TB/s), backwards 84-86 us (537 MB: 6.2-6.4) and 5 us for
// the weight's parts; 32,768 x 4,096 to e4m3 168-170 us (939 MB: 5.5-5.6 TB/s), in single passes up to 197; to int8 178; 16 x 1,024
// 3.7 us, a launch.
#include "pv_rows.h"

#include <algorithm>

using namespace pvo;

namespace {

// An 8-bit format: its largest value, and P values of it from floats that are at most that but for a rounding
struct Fp8 {
    using type = uint8_t;
    static constexpr float MOST = 448.0f;          // (what is nearer to 448 than to 480 rounds to it; NaN stays NaN)
    template <int P> static __device__ void make(const float* v, pack<type, P>& o) {
        if constexpr (P >= 4) {
            uint32_t w[P / 4];
#pragma unroll
            for (int j = 0; j < P; j += 4) {
                int x = __builtin_amdgcn_cvt_pk_fp8_f32(v[j], v[j + 1], 0, false);
                w[j / 4] = __builtin_amdgcn_cvt_pk_fp8_f32(v[j + 2], v[j + 3], x, true);
            }
            __builtin_memcpy(&o, w, P);
        } else {
#pragma unroll
            for (int j = 0; j < P; j++) o.v[j] = type(__builtin_amdgcn_cvt_pk_fp8_f32(v[j], v[j], 0, false));
        }
    }
};
struct Int8 {
    using type = int8_t;
    static constexpr float MOST = 127.0f;
    template <int P> static __device__ void make(const float* v, pack<type, P>& o) {
#pragma unroll
        for (int j = 0; j < P; j++) o.v[j] = v[j] != v[j] ? 0 : type(fminf(fmaxf(rintf(v[j]), -MOST), MOST));
    }
};

template <typename E, typename Q, typename L>
__global__ __launch_bounds__(L::BLOCK) void norm_kernel(const E* __restrict__ x, const E* __restrict__ residual, const float* __restrict__ weight, int64_t N,
                                                        int64_t D, int64_t xs, int64_t rs, float eps, E* __restrict__ y, E* __restrict__ stream,
                                                        float* __restrict__ rstd, typename Q::type* __restrict__ q, float* __restrict__ scale) {
    __shared__ float lds[L::BLOCK / WAVE];
    constexpr int P = 16 / sizeof(E), HELD = L::PACKS ? L::PACKS : 1;
    using pk = pack<E, P>;
    const int lane = threadIdx.x % L::LANES;
    int64_t n = int64_t(blockIdx.x) * L::ROWS + threadIdx.x / L::LANES;
    const bool on = n < N;
    if (!on) n = N - 1;                    // (a workgroup's last rows: computed for the barriers' sake, not stored)
    const E* row = x + n * xs;
    const E* add = residual ? residual + n * rs : nullptr;
    E* const to = stream + n * D;
    const int64_t packs = (D + P - 1) / P;
    pk held[HELD];
    auto each = [&](auto&& f) {            // f(pack, first element's index) over the lane's packs
        if constexpr (L::PACKS) {
#pragma unroll
            for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) f(held[k], i * P);
        } else {
            const E* from = residual ? to : row;
            for (int64_t i = lane; i < packs; i += L::LANES) f(take<P, false>(from, i * P, D), i * P);
        }
    };
    auto join = [&](pk& h, const pk& a, int64_t i) {       // the stream's pack, stored where there is an addition
        if (!add) return;
#pragma unroll
        for (int j = 0; j < P; j++) h.v[j] = E(float(h.v[j]) + float(a.v[j]));
        if (on) leave<false>(h, to, i, D);
    };
    float sum = 0.0f;
    auto square = [&](const pk& h, float m) {
#pragma unroll
        for (int j = 0; j < P; j++) { const float s = m * float(h.v[j]); sum = fmaf(s, s, sum); }
    };
    if constexpr (L::PACKS) {
        pk more[HELD];                     // all loads before the first sum
#pragma unroll
        for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
            held[k] = take<P, true>(row, i * P, D);
            if (add) more[k] = take<P, true>(add, i * P, D);
        }
#pragma unroll
        for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
            join(held[k], more[k], i * P);
            square(held[k], 1.0f);
        }
    } else {
        for (int64_t i = lane; i < packs; i += L::LANES) {
            pk h = take<P, false>(row, i * P, D), a = h;
            if (add) a = take<P, false>(add, i * P, D);
            join(h, a, i * P);
            square(h, 1.0f);
        }
    }
    sum = row_sum<L>(sum, lds);
    // squares that leave 32 bits, or vanish in them where eps does not cover them: once more of m s, which has a square in 32 bits for
    // the largest and for the smallest number of 32 bits alike. (Every lane of a workgroup goes the same way where the sum has a
    // barrier in it: such a workgroup has one row.)
    float m = 1.0f;
    if (sum == INFINITY || (sum < 0x1p-96f && eps < 0x1p-66f)) {
        m = sum < 1.0f ? 0x1p96f : 0x1p-96f;
        sum = 0.0f;
        each([&](const pk& h, int64_t) { square(h, m); });
        sum = row_sum<L>(sum, lds);
    }
    const float r = rsqrtf(sum / float(D) + m * (m * eps));
    if (rstd && on && lane == 0) rstd[n] = m * r;
    if (y) {
        each([&](const pk& h, int64_t i) {
            const auto w = take<P, false>(weight, i, D);
            pk o;
#pragma unroll
            for (int j = 0; j < P; j++) o.v[j] = E(m * float(h.v[j]) * r * w.v[j]);
            if (on) leave<true>(o, y + n * D, i, D);
        });
        return;
    }
    // r is in every y of the row: q = s weight (448 / max |s weight|), and is made from products in two floats (x + the rest of x), so
    // that it is the value nearest to the exact quotient, a tie of which a rounding before would decide by chance. The largest
    // product is found by a key: its bits, which are in order as it is not negative (a NaN being the largest), then its rest's.
    __shared__ unsigned long long keys[L::BLOCK / WAVE];
    unsigned long long key = 0;
    each([&](const pk& h, int64_t i) {
        const auto w = take<P, false>(weight, i, D);
#pragma unroll
        for (int j = 0; j < P; j++) {
            const float a = fabsf(m * float(h.v[j])), b = fabsf(w.v[j]), x = a * b;
            const int32_t rest = __float_as_int(fmaf(a, b, -x));
            const unsigned long long k = uint64_t(__float_as_uint(x)) << 32 | uint32_t(rest ^ (rest >> 31 | INT32_MIN));
            key = k > key ? k : key;
        }
    });
    key = over_row<L>(key, keys, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
    float most = __uint_as_float(uint32_t(key >> 32));
    const int32_t bits = int32_t(uint32_t(key));
    float rest = most < INFINITY ? __int_as_float(bits ^ (~bits >> 31 | INT32_MIN)) : 0.0f;
    if (r == 0.0f) most = NAN;             // an infinity in the row
    if (!on) return;
    if (lane == 0) scale[n] = most / Q::MOST * r;
    const float n2 = most < 0x1p-100f ? 0x1p64f : 1.0f;    // (m n2 itself may be past 32 bits)
    most *= n2;
    rest *= n2;
    const float up = most == 0.0f ? 0.0f : Q::MOST / most;
    const float up_rest = most == 0.0f ? 0.0f : fmaf(-up, rest, fmaf(-up, most, Q::MOST)) / most;
    each([&](const pk& h, int64_t i) {
        const auto w = take<P, false>(weight, i, D);
        float v[P];
#pragma unroll
        for (int j = 0; j < P; j++) {
#pragma clang fp contract(off)     // (y + ... as one operation would count y's own rounding twice)
            const float a = m * float(h.v[j]) * n2, x = a * w.v[j], y = x * up;
            v[j] = y + fmaf(fmaf(a, w.v[j], -x), up, fmaf(x, up_rest, fmaf(x, up, -y)));
        }
        pack<typename Q::type, P> o;
        Q::template make<P>(v, o);
        leave<true>(o, q + n * D, i, D);
    });
}

template <typename E, typename L>
__global__ __launch_bounds__(L::BLOCK) void norm_back_kernel(const E* __restrict__ s, const float* __restrict__ rstd, const float* __restrict__ weight, int64_t N,
                                                             int64_t D, int64_t ss, const E* __restrict__ d_y, const E* __restrict__ d_stream, E* __restrict__ d,
                                                             float* __restrict__ parts) {
    constexpr int P = 16 / sizeof(E), HELD = L::PACKS ? L::PACKS : 1;
    using pk = pack<E, P>;
    __shared__ float lds[L::BLOCK / WAVE];
    const int lane = threadIdx.x % L::LANES, at = threadIdx.x / L::LANES;
    const int64_t packs = (D + P - 1) / P;
    float* part = parts + int64_t(blockIdx.x) * D;
    pack<float, P> w[HELD];
    float dw[HELD][P];
    if constexpr (L::PACKS) {
#pragma unroll
        for (int k = 0; k < HELD; k++) {
            const int64_t i = k * L::LANES + lane;
            w[k] = i < packs ? take<P, false>(weight, i * P, D) : pack<float, P>::load_part(weight, 0);
#pragma unroll
            for (int j = 0; j < P; j++) dw[k][j] = 0.0f;
        }
    } else {
        for (int64_t i = lane; i < D; i += L::LANES) part[i] = 0.0f;
        __syncthreads();
    }
    for (int64_t first = int64_t(blockIdx.x) * L::ROWS; first < N; first += int64_t(gridDim.x) * L::ROWS) {
        const bool on = first + at < N;
        const int64_t n = on ? first + at : N - 1;
        const float r = rstd[n];
        float sum = 0.0f;
        pk u[HELD], dy[HELD], ds[HELD];
        if constexpr (L::PACKS) {
#pragma unroll
            for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
                u[k] = take<P, true>(s + n * ss, i * P, D);
                dy[k] = take<P, true>(d_y + n * D, i * P, D);
                if (d_stream) ds[k] = take<P, true>(d_stream + n * D, i * P, D);
            }
#pragma unroll
            for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
#pragma unroll
                for (int j = 0; j < P; j++) {
                    const float a = float(u[k].v[j]) * r, b = float(dy[k].v[j]);
                    sum = fmaf(b * w[k].v[j], a, sum);
                    if (on) dw[k][j] = fmaf(b, a, dw[k][j]);
                }
            }
        } else {
            for (int64_t i = lane; i < D; i += L::LANES) {
                const float a = float(s[n * ss + i]) * r, b = float(d_y[n * D + i]);
                sum = fmaf(b * weight[i], a, sum);
                if (on) part[i] = fmaf(b, a, part[i]);
            }
        }
        const float mean = row_sum<L>(sum, lds) / float(D);
        if (!on) continue;                 // (the last pass of the loop)
        if constexpr (L::PACKS) {
#pragma unroll
            for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
                pk o;
#pragma unroll
                for (int j = 0; j < P; j++) {
                    const float a = float(u[k].v[j]) * r, g = float(dy[k].v[j]) * w[k].v[j];
                    o.v[j] = E((d_stream ? float(ds[k].v[j]) : 0.0f) + r * (g - a * mean));
                }
                leave<true>(o, d + n * D, i * P, D);
            }
        } else {
            for (int64_t i = lane; i < D; i += L::LANES) {
                const float a = float(s[n * ss + i]) * r, g = float(d_y[n * D + i]) * weight[i];
                d[n * D + i] = E((d_stream ? float(d_stream[n * D + i]) : 0.0f) + r * (g - a * mean));
            }
        }
    }
    if constexpr (L::PACKS) {
        if constexpr (L::ROWS > 1) {       // the rows that the workgroup has at a time: summed by halves, in a fixed order
            __shared__ float sums[L::ROWS / 2][HELD * P][L::LANES];
#pragma unroll
            for (int half = L::ROWS / 2; half; half /= 2) {
                if (at >= half && at < 2 * half) {
#pragma unroll
                    for (int k = 0; k < HELD; k++)
#pragma unroll
                        for (int j = 0; j < P; j++) sums[at - half][k * P + j][lane] = dw[k][j];
                }
                __syncthreads();
                if (at < half) {
#pragma unroll
                    for (int k = 0; k < HELD; k++)
#pragma unroll
                        for (int j = 0; j < P; j++) dw[k][j] += sums[at][k * P + j][lane];
                }
                __syncthreads();
            }
            if (at) return;
        }
#pragma unroll
        for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
            pack<float, P> o;
#pragma unroll
            for (int j = 0; j < P; j++) o.v[j] = dw[k][j];
            leave<false>(o, part, i * P, D);
        }
    }
}

// f(Plan) for rows of D elements of type E: as few lanes as hold the row in one pack each, up to a wave, then more packs, then more
// waves. Backwards, where three tensors, the weights and their gradients' sums are held, 16-bit elements have two packs a lane at
// most; four packs elsewhere, in workgroups as large as the row fills (13,826 x 4,839 float32 by 512 lanes 172 us, by 1,024 195;
// backwards 219 and 243).
template <typename E, bool BACK, typename F> int32_t with_plan(int64_t D, F&& f) {
    constexpr int P = 16 / sizeof(E);
    const int64_t packs = (D + P - 1) / P;
    if (packs <= 8) return f(Plan<8, 1, 32>{});
    if (packs <= 16) return f(Plan<16, 1, 16>{});
    if (packs <= 32) return f(Plan<32, 1, 8>{});
    if (packs <= 64) return f(Plan<64, 1, 4>{});
    if (packs <= 128) return f(Plan<64, 2, 4>{});
    if constexpr (BACK && sizeof(E) == 2) {
        if (packs <= 256) return f(Plan<256, 1, 1>{});
        if (packs <= 512) return f(Plan<256, 2, 1>{});
        if (packs <= 1024) return f(Plan<512, 2, 1>{});
        if (packs <= 2048) return f(Plan<1024, 2, 1>{});
    } else {
        if (packs <= 256) return f(Plan<64, 4, 4>{});
        if (packs <= 512) return f(Plan<256, 2, 1>{});
        if (packs <= 1024) return f(Plan<256, 4, 1>{});
        if (packs <= 2048) return f(Plan<512, 4, 1>{});
        if (packs <= 4096) return f(Plan<1024, 4, 1>{});
    }
    return f(Plan<256, 0, 1>{});
}

template <typename E> int rows_of(int64_t D) {
    int rows = 0;
    with_plan<E, true>(D, [&](auto plan) { rows = decltype(plan)::ROWS; return 0; });
    return rows;
}

int32_t check(int64_t N, int64_t D, int32_t dtype, char* err, size_t cap) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, cap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (N < 0 || D < 1 || N > INT32_MAX) return fail(PV_EARG, err, cap, "shape: 0 <= N < 2^31, D >= 1");
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
        return with_plan<E, false>(D, [&](auto plan) {
            using L = decltype(plan);
            constexpr int64_t MOST = (MOST_ITEMS - 1) / L::BLOCK * L::ROWS;    // rows of a launch
            const auto from = [](auto* p, int64_t i) { return p ? p + i : nullptr; };
            for (int64_t n = 0; n < N; n += MOST) {
                const int64_t rows = std::min(N - n, MOST);
                norm_kernel<E, Q, L><<<dim3((rows + L::ROWS - 1) / L::ROWS), L::BLOCK, 0, hipStream_t(stream)>>>(
                    static_cast<const E*>(x) + n * xs, from(static_cast<const E*>(residual), n * rs), weight, rows, D, xs, rs, eps, from(static_cast<E*>(y), n * D),
                    from(static_cast<E*>(stream_out), n * D), from(rstd, n), from(static_cast<typename Q::type*>(q), n * D), from(scale, n));
            }
            return launched(err, errcap);
        });
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

uint64_t pv_add_rms_norm_work_bytes(int64_t N, int64_t D) {
    // (of either element size's plan: the one with fewer rows in a workgroup has more parts)
    const int64_t g = N > 0 && D > 0 ? std::max(groups_of(N, rows_of<float>(D)), groups_of(N, rows_of<bf16>(D))) : 0;
    return g > 1 ? uint64_t(g) * uint64_t(D) * 4 : 0;
}

int32_t pv_add_rms_norm_backward_hip(const void* s, const float* rstd, const float* weight, int64_t N, int64_t D, int64_t s_row, const void* d_y,
                                     const void* d_stream, int32_t dtype, void* d, float* d_weight, void* work, uint64_t work_bytes, void* stream, char* err,
                                     size_t errcap) {
    if (int32_t e = check(N, D, dtype, err, errcap)) return e;
    if (!d_weight || (N && (!s || !rstd || !weight || !d_y || !d))) return fail(PV_EARG, err, errcap, "null argument");
    const uint64_t need = pv_add_rms_norm_work_bytes(N, D);
    if (need && (!work || work_bytes < need || !aligned(work, 16))) return fail(PV_EARG, err, errcap, "work: too small, or not 16-byte aligned");
    const hipStream_t st = hipStream_t(stream);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        return with_plan<E, true>(D, [&](auto plan) {
            using L = decltype(plan);
            const int64_t g = groups_of(N, L::ROWS);
            float* parts = g > 1 ? static_cast<float*>(work) : d_weight;       // (one workgroup's part is the sum)
            if (N) norm_back_kernel<E, L><<<dim3(g), L::BLOCK, 0, st>>>(static_cast<const E*>(s), rstd, weight, N, D, s_row, static_cast<const E*>(d_y),
                                                                        static_cast<const E*>(d_stream), static_cast<E*>(d), parts);
            constexpr int64_t MOST = MOST_ITEMS / END_WAVES / 2;               // columns of a launch
            for (int64_t i = 0; g != 1 && i < D; i += MOST)
                norm_weight_kernel<<<dim3((std::min(D - i, MOST) + WAVE - 1) / WAVE), END_WAVES * WAVE, 0, st>>>(parts, g, D, i, d_weight, nullptr);
            return launched(err, errcap);
        });
    });
}

}  // extern "C"
