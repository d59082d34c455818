// The residual stream's addition with dropout of what is added, its layer norm, and the gradients.
//
//   s = residual + drop(x), rounded to the stream's type: what the next layer adds to, and what is normalised
//   y = (s - mean) r weight + bias,  r = 1 / sqrt(var + eps), mean and var over the row
//   backward, with u = (s - mean) r and g = d_y weight:  d = d_stream + r (g - mean(g) - u mean(g u)), the residual's gradient;
//   d_x = drop(d);  d_weight = sum over rows of d_y u;  d_bias = sum over rows of d_y
//
// As in pv_norm.hip a row's elements stay in registers between its sums and its outputs, so every byte is read once and written
// once; dropped places are made again from their index (pv_drop.h) and not stored. The variance is that of s - mean, by a second
// sum over the registers; a third one, of s - mean itself, takes out what the first mean was off by, so that rows far from zero
// lose nothing but what their elements' own type has lost. Sums in 32 bits.
//
// What bounds it: the bytes. bfloat16, 65,536 x 1,024, with dropout: 90-99 us (5.4-6.0 TB/s) and 120-129 backwards (5.2-5.6), with 5 for the
// sums of the partial rows; float16 without, 32,768 x 4,096: 170-174 us (6.2).
#include "pv_drop.h"
#include "pv_rows.h"

#include <algorithm>

using namespace pvo;

namespace {

// Two sums over the lanes of a row at once
struct Two { float a, b; };
template <typename L> __device__ inline Two row_sums(Two x, Two* lds) {
#pragma unroll
    for (int d = (L::LANES < WAVE ? L::LANES : WAVE) / 2; d; d >>= 1) x = {x.a + __shfl_xor(x.a, d, WAVE), x.b + __shfl_xor(x.b, d, WAVE)};
    if constexpr (L::WAVES > 1) {
        const int row = threadIdx.x / L::LANES, wave = threadIdx.x / WAVE;
        __syncthreads();                   // the last use of lds is over
        if (threadIdx.x % WAVE == 0) lds[wave] = x;
        __syncthreads();
        x = lds[row * L::WAVES];
#pragma unroll
        for (int w = 1; w < L::WAVES; w++) x = {x.a + lds[row * L::WAVES + w].a, x.b + lds[row * L::WAVES + w].b};
    }
    return x;
}

// What the backward pass takes of a row: half its mean, in two floats, and twice r. (Of halves, so that the difference of numbers
// at the ends of the type's range stays inside it.)
struct Stats { float half, rest, twice; };
__device__ inline float unit_of(float s, Stats q) { return (fmaf(s, 0.5f, -q.half) - q.rest) * q.twice; }

template <typename E, typename L, bool DROP>
__global__ __launch_bounds__(L::BLOCK) void layer_kernel(const E* __restrict__ x, const E* __restrict__ residual, const float* __restrict__ weight,
                                                         const float* __restrict__ bias, int64_t N, int64_t D, int64_t xs, int64_t rs, float eps, int64_t row0,
                                                         Drop drop, E* __restrict__ y, E* __restrict__ stream, Stats* __restrict__ stats) {
    __shared__ Two lds[L::BLOCK / WAVE];
    constexpr int P = 16 / sizeof(E), HELD = L::PACKS ? L::PACKS : 1;
    using pk = pack<E, P>;
    const int lane = threadIdx.x % L::LANES;
    int64_t n = int64_t(blockIdx.x) * L::ROWS + threadIdx.x / L::LANES;
    const bool on = n < N;
    if (!on) n = N - 1;                    // (a workgroup's last rows: computed for the barriers' sake, not stored)
    const E* row = x + n * xs;
    const E* add = residual ? residual + n * rs : nullptr;
    E* const to = stream ? stream + n * D : nullptr;
    const int64_t packs = (D + P - 1) / P;
    pk held[HELD];
    auto each = [&](auto&& f) {            // f(pack, first element's index) over the lane's packs
        if constexpr (L::PACKS) {
#pragma unroll
            for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) f(held[k], i * P);
        } else {
            const E* from = stream ? to : row;
            for (int64_t i = lane; i < packs; i += L::LANES) f(take<P, false>(from, i * P, D), i * P);
        }
    };
    uint64_t seed = 0;
    if constexpr (DROP) seed = drop.seed();
    auto join = [&](pk& h, const pk& a, int64_t i) {       // the stream's pack, stored where it is not x itself
        if constexpr (DROP) {
            float v[P];
            each_kept<P>(drop, seed, uint64_t(row0 + n) * uint64_t(D) + uint64_t(i), [&](int j, bool kept) { v[j] = kept ? float(h.v[j]) * drop.up : 0.0f; });
#pragma unroll
            for (int j = 0; j < P; j++) h.v[j] = E(add ? v[j] + float(a.v[j]) : v[j]);
        } else if (add) {
#pragma unroll
            for (int j = 0; j < P; j++) h.v[j] = E(float(h.v[j]) + float(a.v[j]));
        }
        if (to && on) leave<false>(h, to, i, D);
    };
    // elements behind the row's end are 0 in a pack, and have no part in sums around a mean
    float m = 1.0f;
    Two sum = {0.0f, 0.0f};
    auto plain = [&](const pk& h) {
#pragma unroll
        for (int j = 0; j < P; j++) sum.a = fmaf(m, float(h.v[j]), sum.a);
    };
    float mean = 0.0f;
    auto around = [&](const pk& h, int64_t i) {
#pragma unroll
        for (int j = 0; j < P; j++) {
            const float d = i + j < D ? fmaf(m, float(h.v[j]), -mean) : 0.0f;
            sum.a += d;
            sum.b = fmaf(d, d, sum.b);
        }
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
            plain(held[k]);
        }
    } else {
        for (int64_t i = lane; i < packs; i += L::LANES) {
            pk h = take<P, false>(row, i * P, D), a = h;
            if (add) a = take<P, false>(add, i * P, D);
            join(h, a, i * P);
            plain(h);
        }
    }
    const float share = 1.0f / float(D);
    auto spread = [&] {                    // the row's mean, then what that is off by and the squares around it
        sum = row_sums<L>(sum, lds);
        mean = sum.a * share;
        sum = {0.0f, 0.0f};
        each([&](const pk& h, int64_t i) { around(h, i); });
        sum = row_sums<L>(sum, lds);
    };
    spread();
    float off = sum.a * share, var = fmaxf(fmaf(sum.b, share, -off * off), 0.0f);
    if (sum.b != sum.b) var = sum.b;
    // sums that leave 32 bits, or squares that vanish in them where eps does not cover them: once more of m s. (Every lane of a
    // workgroup goes the same way where the sum has a barrier in it: such a workgroup has one row.)
    const bool high = !(sum.b < INFINITY), low = var < 0x1p-96f && eps < 0x1p-66f && fabsf(mean) < 0x1p-30f;
    if (high || low) {
        m = high ? 0x1p-96f : 0x1p96f;
        sum = {0.0f, 0.0f};
        each([&](const pk& h, int64_t) { plain(h); });
        spread();
        off = sum.a * share;
        var = fmaxf(fmaf(sum.b, share, -off * off), 0.0f);
        if (sum.b != sum.b) var = sum.b;
    }
    // (of elements that are all alike nothing but eps is left, which may have vanished with m)
    const float more = m * (m * eps), r = var + more == 0.0f && eps != 0.0f ? rsqrtf(eps) / m : rsqrtf(var + more);
    if (stats && on && lane == 0) stats[n] = {0.5f * (mean / m), 0.5f * (off / m), 2.0f * (m * r)};
    each([&](const pk& h, int64_t i) {
        const auto w = take<P, false>(weight, i, D);
        auto b = w;
        if (bias) b = take<P, false>(bias, i, D);
        pk o;
#pragma unroll
        for (int j = 0; j < P; j++) {
            const float u = (fmaf(m, float(h.v[j]), -mean) - off) * r;
            o.v[j] = E(bias ? fmaf(u, w.v[j], b.v[j]) : u * w.v[j]);
        }
        if (on) leave<true>(o, y + n * D, i, D);
    });
}

template <typename E, typename L, bool DROP>
__global__ __launch_bounds__(L::BLOCK) void layer_back_kernel(const E* __restrict__ s, const Stats* __restrict__ stats, const float* __restrict__ weight, int64_t N,
                                                              int64_t D, int64_t ss, const E* __restrict__ d_y, const E* __restrict__ d_stream, Drop drop,
                                                              E* __restrict__ d, E* __restrict__ d_x, float* __restrict__ weight_parts,
                                                              float* __restrict__ bias_parts) {
    constexpr int P = 16 / sizeof(E), HELD = L::PACKS ? L::PACKS : 1;
    using pk = pack<E, P>;
    __shared__ Two lds[L::BLOCK / WAVE];
    const int lane = threadIdx.x % L::LANES, at = threadIdx.x / L::LANES;
    const int64_t packs = (D + P - 1) / P;
    float *part_w = weight_parts + int64_t(blockIdx.x) * D, *part_b = bias_parts + int64_t(blockIdx.x) * D;
    const float share = 1.0f / float(D);
    uint64_t seed = 0;
    if constexpr (DROP) seed = drop.seed();
    float dw[HELD][P], db[HELD][P];
    if constexpr (L::PACKS) {
#pragma unroll
        for (int k = 0; k < HELD; k++)
#pragma unroll
            for (int j = 0; j < P; j++) dw[k][j] = db[k][j] = 0.0f;
    } else {
        for (int64_t i = lane; i < D; i += L::LANES) part_w[i] = part_b[i] = 0.0f;
        __syncthreads();
    }
    auto write = [&](const float(&v)[P], int64_t n, int64_t i) {
        pk o;
#pragma unroll
        for (int j = 0; j < P; j++) o.v[j] = E(v[j]);
        leave<true>(o, d + n * D, i, D);
        if constexpr (DROP) {
            each_kept<P>(drop, seed, uint64_t(n) * uint64_t(D) + uint64_t(i), [&](int j, bool kept) { o.v[j] = kept ? E(v[j] * drop.up) : E(0.0f); });
            leave<true>(o, d_x + n * D, i, D);
        }
    };
    for (int64_t first = int64_t(blockIdx.x) * L::ROWS; first < N; first += int64_t(gridDim.x) * L::ROWS) {
        const bool on = first + at < N;
        const int64_t n = on ? first + at : N - 1;
        const Stats q = stats[n];
        const float r = 0.5f * q.twice;
        Two sum = {0.0f, 0.0f};
        pk u[HELD], dy[HELD], ds[HELD];
        auto gather = [&](int k, float a, float b, float w, int j) {
            sum.a = fmaf(b, w, sum.a);
            sum.b = fmaf(b * w, a, sum.b);
        };
        if constexpr (L::PACKS) {
#pragma unroll
            for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
                u[k] = take<P, true>(s + n * ss, i * P, D);
                dy[k] = take<P, true>(d_y + n * D, i * P, D);
                if (d_stream) ds[k] = take<P, true>(d_stream + n * D, i * P, D);
            }
#pragma unroll
            for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
                const auto w = take<P, false>(weight, i * P, D);
#pragma unroll
                for (int j = 0; j < P; j++) {
                    const float a = unit_of(float(u[k].v[j]), q), b = float(dy[k].v[j]);
                    gather(k, a, b, w.v[j], j);
                    if (on) { dw[k][j] = fmaf(b, a, dw[k][j]); db[k][j] += b; }
                }
            }
        } else {
            for (int64_t i = lane; i < D; i += L::LANES) {
                const float a = unit_of(float(s[n * ss + i]), q), b = float(d_y[n * D + i]);
                gather(0, a, b, weight[i], 0);
                if (on) { part_w[i] = fmaf(b, a, part_w[i]); part_b[i] += b; }
            }
        }
        sum = row_sums<L>(sum, lds);
        sum.a *= share;
        sum.b *= share;
        if (!on) continue;                 // (the last pass of the loop)
        if constexpr (L::PACKS) {
#pragma unroll
            for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
                const auto w = take<P, false>(weight, i * P, D);
                float o[P];
#pragma unroll
                for (int j = 0; j < P; j++) {
                    const float a = unit_of(float(u[k].v[j]), q);
                    o[j] = fmaf(r, fmaf(-a, sum.b, fmaf(float(dy[k].v[j]), w.v[j], -sum.a)), d_stream ? float(ds[k].v[j]) : 0.0f);
                }
                write(o, n, i * P);
            }
        } else {
            for (int64_t i = lane; i < packs; i += L::LANES) {
                const auto w = take<P, false>(weight, i * P, D);
                const pk v = take<P, false>(s + n * ss, i * P, D), g = take<P, false>(d_y + n * D, i * P, D);
                pk more = g;
                if (d_stream) more = take<P, false>(d_stream + n * D, i * P, D);
                float o[P];
#pragma unroll
                for (int j = 0; j < P; j++) {
                    const float a = unit_of(float(v.v[j]), q);
                    o[j] = fmaf(r, fmaf(-a, sum.b, fmaf(float(g.v[j]), w.v[j], -sum.a)), d_stream ? float(more.v[j]) : 0.0f);
                }
                write(o, n, i * P);
            }
        }
    }
    if constexpr (L::PACKS) {
        if constexpr (L::ROWS > 1) {       // the rows that the workgroup has at a time: summed by halves, in a fixed order
            __shared__ float sums[L::ROWS / 2][HELD * P][L::LANES];
            auto fold = [&](float(&v)[HELD][P]) {
#pragma unroll
                for (int half = L::ROWS / 2; half; half /= 2) {
                    if (at >= half && at < 2 * half) {
#pragma unroll
                        for (int k = 0; k < HELD; k++)
#pragma unroll
                            for (int j = 0; j < P; j++) sums[at - half][k * P + j][lane] = v[k][j];
                    }
                    __syncthreads();
                    if (at < half) {
#pragma unroll
                        for (int k = 0; k < HELD; k++)
#pragma unroll
                            for (int j = 0; j < P; j++) v[k][j] += sums[at][k * P + j][lane];
                    }
                    __syncthreads();
                }
            };
            fold(dw);
            fold(db);
            if (at) return;
        }
#pragma unroll
        for (int k = 0; k < HELD; k++) if (const int64_t i = k * L::LANES + lane; i < packs) {
            pack<float, P> o;
#pragma unroll
            for (int j = 0; j < P; j++) o.v[j] = dw[k][j];
            leave<false>(o, part_w, i * P, D);
#pragma unroll
            for (int j = 0; j < P; j++) o.v[j] = db[k][j];
            leave<false>(o, part_b, i * P, D);
        }
    }
}

// f(Plan) for rows of D elements of type E, as in pv_norm.hip: as few lanes as hold the row in one pack each, up to a wave, then more
// packs, then more waves. Backwards, with two rows of sums beside the three tensors, a lane has two packs at most.
template <typename E, bool BACK, typename F> int32_t with_plan(int64_t D, F&& f) {
    constexpr int P = 16 / sizeof(E);
    const int64_t packs = (D + P - 1) / P;
    if (packs <= 8) return f(Plan<8, 1, 32>{});
    if (packs <= 16) return f(Plan<16, 1, 16>{});
    if (packs <= 32) return f(Plan<32, 1, 8>{});
    if (packs <= 64) return f(Plan<64, 1, 4>{});
    if (packs <= 128) return f(Plan<64, 2, 4>{});
    if constexpr (BACK) {
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

int32_t check(int64_t N, int64_t D, double p, int32_t dtype, char* err, size_t cap) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, cap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (N < 0 || D < 1 || N > INT32_MAX || D > INT32_MAX) return fail(PV_EARG, err, cap, "shape: 0 <= N < 2^31, 1 <= D < 2^31");
    if (const char* m = drop_error(p)) return fail(PV_EARG, err, cap, m);
    return PV_OK;
}

// f(true or false) as a type, by whether anything is dropped
template <typename F> int32_t with_drop(const Drop& drop, F&& f) { return drop.least ? f(std::true_type{}) : f(std::false_type{}); }

}  // namespace

extern "C" {

int32_t pv_add_layer_norm_hip(const void* x, const void* residual, const float* weight, const float* bias, int64_t N, int64_t D, int64_t x_row,
                              int64_t residual_row, float eps, double p, const int64_t* seed_at, int64_t seed, uint32_t site, int32_t dtype, void* y, void* stream_out,
                              float* stats, void* stream, char* err, size_t errcap) {
    if (int32_t e = check(N, D, p, dtype, err, errcap)) return e;
    if (!N) return PV_OK;
    const Drop drop = drop_of(seed_at, seed, site, p);
    if (!x || !weight || !y || ((residual || drop.least) && !stream_out)) return fail(PV_EARG, err, errcap, "null argument");
    if (!aligned(seed_at, 8)) return fail(PV_EARG, err, errcap, "seed: not a multiple of 8 as an address");
    const bool kept = residual || drop.least;
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        return with_plan<E, false>(D, [&](auto plan) {
            return with_drop(drop, [&](auto dropped) {
                using L = decltype(plan);
                constexpr int64_t MOST = (MOST_ITEMS - 1) / L::BLOCK * L::ROWS;    // rows of a launch
                const auto from = [](auto* p, int64_t i) { return p ? p + i : nullptr; };
                for (int64_t n = 0; n < N; n += MOST) {
                    const int64_t rows = std::min(N - n, MOST);
                    layer_kernel<E, L, decltype(dropped)::value><<<dim3((rows + L::ROWS - 1) / L::ROWS), L::BLOCK, 0, hipStream_t(stream)>>>(
                        static_cast<const E*>(x) + n * x_row, from(static_cast<const E*>(residual), n * residual_row), weight, bias, rows, D, x_row, residual_row, eps, n,
                        drop, static_cast<E*>(y) + n * D, kept ? static_cast<E*>(stream_out) + n * D : nullptr, from(reinterpret_cast<Stats*>(stats), n));
                }
                return launched(err, errcap);
            });
        });
    });
}

uint64_t pv_add_layer_norm_work_bytes(int64_t N, int64_t D) {
    // (of either element size's plan: the one with fewer rows in a workgroup has more parts)
    const int64_t g = N > 0 && D > 0 ? std::max(groups_of(N, rows_of<float>(D)), groups_of(N, rows_of<bf16>(D))) : 0;
    return g > 1 ? uint64_t(g) * uint64_t(D) * 8 : 0;
}

int32_t pv_add_layer_norm_backward_hip(const void* s, const float* stats, const float* weight, int64_t N, int64_t D, int64_t s_row, const void* d_y,
                                       const void* d_stream, double p, const int64_t* seed_at, int64_t seed, uint32_t site, int32_t dtype, void* d, void* d_x,
                                       float* d_weight, float* d_bias, void* work, uint64_t work_bytes, void* stream, char* err, size_t errcap) {
    if (int32_t e = check(N, D, p, dtype, err, errcap)) return e;
    const Drop drop = drop_of(seed_at, seed, site, p);
    if (!d_weight || !d_bias || (N && (!s || !stats || !weight || !d_y || !d || (drop.least && !d_x)))) return fail(PV_EARG, err, errcap, "null argument");
    if (!aligned(seed_at, 8)) return fail(PV_EARG, err, errcap, "seed: not a multiple of 8 as an address");
    const uint64_t need = pv_add_layer_norm_work_bytes(N, D);
    if (need && (!work || work_bytes < need || !aligned(work, 16))) return fail(PV_EARG, err, errcap, "work: too small, or not 16-byte aligned");
    const hipStream_t st = hipStream_t(stream);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        return with_plan<E, true>(D, [&](auto plan) {
            return with_drop(drop, [&](auto dropped) {
                using L = decltype(plan);
                const int64_t g = groups_of(N, L::ROWS);
                float* parts_w = g > 1 ? static_cast<float*>(work) : d_weight;     // (one workgroup's part is the sum)
                float* parts_b = g > 1 ? static_cast<float*>(work) + g * D : d_bias;
                if (N)
                    layer_back_kernel<E, L, decltype(dropped)::value><<<dim3(g), L::BLOCK, 0, st>>>(static_cast<const E*>(s), reinterpret_cast<const Stats*>(stats),
                                                                                                   weight, N, D, s_row, static_cast<const E*>(d_y),
                                                                                                   static_cast<const E*>(d_stream), drop, static_cast<E*>(d),
                                                                                                   static_cast<E*>(d_x), parts_w, parts_b);
                constexpr int64_t MOST = MOST_ITEMS / END_WAVES / 4;               // columns of a launch
                for (int64_t i = 0; g != 1 && i < D; i += MOST) {
                    const dim3 grid((std::min(D - i, MOST) + WAVE - 1) / WAVE, 2);
                    norm_weight_kernel<<<grid, END_WAVES * WAVE, 0, st>>>(parts_w, g, D, i, d_weight, d_bias);
                }
                return launched(err, errcap);
            });
        });
    });
}

}  // extern "C"
