// The head and loss of a model that predicts the next token of a window over a small alphabet, and the gradients.
//
//   logits[b, t, v] = hidden[b, t, :] . weight[v, :];  a place (b, t) counts if tokens[b, t + 1] is one of the V ids and not
//   `ignore` (the last place of a row never does);  each = logsumexp(logits) - logits[tokens[b, t + 1]], 0 where nothing
//   counts;  loss = sum of each / number of places that count (0 where there are none)
//   d_logits = (softmax - onehot) * w, w = scale / count or the place's own factor;
//   d_hidden = d_logits weight (0 where a place does not count);  d_weight = sum over places of d_logits^T hidden
// What stands in hidden at places that do not count (NaN too) reaches nothing.
//
// The alphabet fills one 16-wide matrix tile. A tile of 16 places goes through it three times: logits = weight hidden^T
// (contracted over D), d_hidden = weight^T d_logits (over the ids), d_weight = hidden^T d_logits (over the places). A wave has
// a slab of columns and keeps there, in registers, the weights in both operands' layouts, the tile's hidden values and the sums
// of d_weight: `fused_kernel` reads hidden once for all three, with one exchange of partial logits between the waves of a
// workgroup a tile. Rows of more slabs than a workgroup has waves go through `place_kernel` (logits, d_logits stored) and
// `grad_kernel` (the other two by columns), which reads hidden again.
// The operand that a product needs transposed is made by a product with the identity, which is exact.
//   H2  hidden and weight alike in bfloat16 or float16: products of such numbers, sums in 32 bits; d_logits as the sum of three of
//       them, which is all of its 24 bits
//   F3  weight in float32: values in 32 bits, 32-bit products
//
// What bounds it: the bytes where only losses are asked for (16 x 32,768 x 512 bfloat16 95-97 us, 537 MB: 5.5-5.7 TB/s; float32
// 195 us, 1.07 GB: 5.5; bfloat16 with weight in float32 191 us: 2.8, half of it the products). With gradients each tile is a chain
// of three products, an exchange and a softmax, every wave doing the softmax again for itself; 16 waves a CU overlap it with the
// loads and stores: 8 x 8,192 x 1,024 bfloat16 63-65 us (268 MB: 4.1-4.2 TB/s) and 10 us for the count before and the parts of
// d_weight after it. F3 is the same chain with products at an eighth of bfloat16's rate, which by their count alone would be some
// 58 us there: float32 152 us with the launches beside it (3.5 TB/s), bfloat16 with weight in float32 128 (2.1; all in float16 79,
// bfloat16 73). 5 x 2,049 x 500 float32, one or two tiles a workgroup, 22 us and 8: latency.
#include "pv_ops.h"

#include <algorithm>

using namespace pvo;

namespace {

constexpr int VMAX = 16;                   // ids at most
constexpr int TILE = 16;                   // places of a tile
constexpr int COUNTS = 256;                // workgroups that count places
constexpr int BLOCK = 256;
constexpr int MOST_WAVES = 16;             // of a workgroup
constexpr int END_WAVES = 16;
// of a row: end_kernel has END_WAVES work items for each element of the head, and one workgroup more
constexpr int64_t MOST_COLUMNS = 1 << 23;
static_assert(MOST_COLUMNS * VMAX * END_WAVES + END_WAVES * 64 < MOST_ITEMS, "a launch's work items");

using f32x4 = __attribute__((ext_vector_type(4))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;

struct Shape {
    int64_t B, T, D, N, hb, ht, tb;        // N = B T; strides in elements: hidden (batch, time), tokens (batch)
    int64_t ignore, Dp;                    // Dp: D filled up to whole slabs
    int32_t V, token_bytes;
    bool flat;                             // hidden's places are ht apart throughout
};

// What the matrix instructions hold in a lane: l = 16 g + c. First operand: row c, elements k of its group g; second: column
// c, the same k; result: column c, rows 4 g + r. k is 8 g + j for 16x16x32, 4 g + j for 16x16x16, g for 16x16x4.
__device__ inline int lane_c() { return threadIdx.x % 16; }
__device__ inline int lane_g() { return threadIdx.x % WAVE / 16; }

// A pack of which `left` elements are in the row: all, some, or none
template <typename E, int N> __device__ inline pack<E, N> get(const E* p, int64_t left) {
    return left >= N ? pack<E, N>::load(p) : pack<E, N>::load_part(p, left);
}
template <typename E, int N> __device__ inline void put(const pack<E, N>& v, E* p, int64_t left) {
    if (left >= N) v.store(p); else v.store_part(p, left);
}
// f(true) for a slab that lies within the row, else f(false): asked once, not at each load
template <typename F> __device__ inline void over_slab(bool within, F&& f) {
    if (within) f(std::true_type{}); else f(std::false_type{});
}

// x joined with the values of the lanes of the same c (l ^ 16, l ^ 32, l ^ 48)
template <typename F> __device__ inline float over_groups(float x, F&& join) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = join(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return join(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// The products of 16-bit operands, with sums in 32 bits
template <typename E> struct Half {
    using x4 = __attribute__((ext_vector_type(4))) E;
    using x8 = __attribute__((ext_vector_type(8))) E;
    static __device__ f32x4 product(x4 a, x4 b, f32x4 c) {             // 16 x 16 x 16
        if constexpr (std::is_same_v<E, bf16>) return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
    }
    static __device__ f32x4 product(x8 a, x8 b, f32x4 c) {             // 16 x 16 x 32
        if constexpr (std::is_same_v<E, bf16>) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// A slab of 128 columns in bfloat16 or float16. The gradients of the logits go into products as the sum of three such numbers. In
// float16, whose exponents are few, powers of two bring them near its largest number first: a place's own for d_hidden, and for
// d_weight one for all that the wave has summed up, which grows (with the sums rescaled) when a tile needs it.
template <typename E_> struct H2 {
    using E = E_;
    using K = E_;                          // what the weights are laid out as
    using x4 = typename Half<E>::x4;
    using x8 = typename Half<E>::x8;
    static constexpr bool SCALED = std::is_same_v<E, f16>;
    static constexpr int COLS = 128, STEPS = 4, TILES = 8;
    struct Rows { x8 h[STEPS]; };          // column 32 q + 8 g + j of place c
    struct Sums { f32x4 dw[TILES]; int e; };                  // id c, columns 32 q + 8 g + 4 t + r at 2 q + t (SCALED: over 2^(e - 15))
    x8 w[STEPS];                           // id c, columns as Rows
    using Back = x4;
    const Back* wt;                        // [TILES][lanes], in LDS: column 32 q + 8 (c / 4) + 4 t + c % 4 at 2 q + t, ids 4 g + j

    __device__ void weights(const K* wr, int64_t Dp, int64_t c0) {
#pragma unroll
        for (int q = 0; q < STEPS; q++) w[q] = *reinterpret_cast<const x8*>(wr + lane_c() * Dp + c0 + 32 * q + 8 * lane_g());
    }
    // (to: the wave's own room, so no other wave waits for it)
    __device__ void weights_back(const K* wc, int64_t c0, Back* to) {
        const int c = lane_c();
        to += threadIdx.x % WAVE;
#pragma unroll
        for (int k = 0; k < TILES; k++)
            to[k * WAVE] = *reinterpret_cast<const Back*>(wc + (c0 + 32 * (k / 2) + 8 * (c / 4) + 4 * (k % 2) + c % 4) * VMAX + 4 * lane_g());
        wt = to;
    }
    static __device__ Rows rows(const E* row, int64_t c0, int64_t D) {
        Rows R;
        row += c0 + 8 * lane_g();
        over_slab(c0 + COLS <= D, [&](auto whole) {
#pragma unroll
            for (int q = 0; q < STEPS; q++) {
                const auto p = whole ? pack<E, 8>::load(row + 32 * q) : get<E, 8>(row + 32 * q, D - c0 - 32 * q - 8 * lane_g());
                __builtin_memcpy(&R.h[q], &p, 16);
            }
        });
        return R;
    }
    static __device__ void clear(Rows& R) {
#pragma unroll
        for (int q = 0; q < STEPS; q++)
#pragma unroll
            for (int j = 0; j < 8; j++) R.h[q][j] = E(0.0f);
    }
    __device__ f32x4 logits(const Rows& R, f32x4 l) const {
#pragma unroll
        for (int q = 0; q < STEPS; q++) l = Half<E>::product(w[q], R.h[q], l);
        return l;
    }
    static __device__ x4 rounded(f32x4 x) { return __builtin_convertvector(x, x4); }
    // A right operand as the sum of its parts, a product of 16 each, the smallest first. (The sum goes through products of one
    // shape: a 16 x 16 x 16 product's sum taken up by a 16 x 16 x 32 one right behind it lost rows, the compiler leaving no wait.)
    struct Parts {
        x4 part[3];
        static __device__ Parts of(f32x4 x) {
            Parts p;
#pragma unroll
            for (int k = 0; k < 3; k++) {
                p.part[k] = rounded(x);
                x -= __builtin_convertvector(p.part[k], f32x4);
            }
            return p;
        }
        // by the identity: rows to columns
        __device__ Parts turned(x4 one) const {
            Parts p;
#pragma unroll
            for (int k = 0; k < 3; k++) p.part[k] = rounded(Half<E>::product(part[k], one, f32x4{0.0f, 0.0f, 0.0f, 0.0f}));
            return p;
        }
        __device__ f32x4 product(x4 left, f32x4 c) const {
#pragma unroll
            for (int k = 2; k >= 0; k--) c = Half<E>::product(left, part[k], c);
            return c;
        }
    };
    static __device__ f32x4 times(f32x4 x, int e) {
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = ldexpf(x[r], e);
        return x;
    }
    // dl: d_logits of place c, ids 4 g + j
    __device__ void back(const Rows& R, f32x4 dl, E* d_row, int64_t c0, int64_t D, bool store, Sums& S) const {
        const int c = lane_c(), g = lane_g();
        const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
        x4 one;                            // the identity, 16 x 16
#pragma unroll
        for (int j = 0; j < 4; j++) one[j] = E(c == 4 * g + j ? 1.0f : 0.0f);
        int e = 0;                         // d_hidden is made of 2^(15 - e) d_logits
        if constexpr (SCALED) {
            float most = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) most = fabsf(dl[j]) < INFINITY ? fmaxf(most, fabsf(dl[j])) : most;
            most = over_groups(most, [](float a, float b) { return fmaxf(a, b); });
            e = int(__float_as_uint(fmaxf(most, 0x1p-100f)) >> 23) - 126;
            int all = e;
#pragma unroll
            for (int d = 1; d < TILE; d *= 2) all = max(all, __shfl_xor(all, d, WAVE));
            all = __builtin_amdgcn_readfirstlane(all);
            if (all > S.e) {
#pragma unroll
                for (int k = 0; k < TILES; k++) S.dw[k] = times(S.dw[k], S.e - all);
                S.e = all;
            }
        }
        const Parts p = Parts::of(SCALED ? times(dl, 15 - e) : dl);
        const bool whole = c0 + COLS <= D;
        d_row += c0 + 8 * g;
#pragma unroll
        for (int q = 0; q < STEPS; q++) {
            x4 o[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {  // (every lane's weights are operands, whether it stores or not)
                f32x4 x = p.product(wt[(2 * q + t) * WAVE], none);
                if constexpr (SCALED) x = times(x, e - 15);
                o[t] = rounded(x);
            }
            if (store) {
                pack<E, 8> row;
                __builtin_memcpy(&row, o, 16);
                if (whole) row.store(d_row + 32 * q);          // (past the caches, rows that are not whole lines take half as long again: 65,536 x 1,000 in 117 us instead of 78)
                else put<E, 8>(row, d_row + 32 * q, D - c0 - 32 * q - 8 * g);
            }
        }
        // Id c, places 4 g + j. (After d_hidden: with both operands' parts held at once registers were spilled, and 8 x 8,192 x 1,024
        // took 80 us instead of 73 in bfloat16, 95 instead of 79 in float16.)
        const Parts turned = (SCALED ? Parts::of(times(dl, 15 - S.e)) : p).turned(one);
#pragma unroll
        for (int k = 0; k < TILES; k++) {
            x4 h;                          // column 32 q + 8 g + 4 t + j of place c; turned: column 32 q + 8 (c / 4) + 4 t + c % 4, places 4 g + j
#pragma unroll
            for (int j = 0; j < 4; j++) h[j] = R.h[k / 2][4 * (k % 2) + j];
            S.dw[k] = turned.product(rounded(Half<E>::product(h, one, none)), S.dw[k]);
        }
    }
    static __device__ void begin(Sums& S) { S = {}; S.e = -99; }
    static __device__ f32x4 end(const Sums& S, int k) { return SCALED ? times(S.dw[k], S.e - 15) : S.dw[k]; }
    // where the columns of result k's rows 4 g + r begin
    static __device__ int column(int k) { return 32 * (k / 2) + 8 * lane_g() + 4 * (k % 2); }
};

// A slab of 64 columns in 32 bits
template <typename E_> struct F3 {
    using E = E_;
    using K = float;
    static constexpr int COLS = 64, STEPS = 4, TILES = 4;
    struct Rows { pack<E, 4> h[STEPS]; };  // column 16 s + 4 g + j of place c
    struct Sums { f32x4 dw[TILES]; };      // id c, columns 16 s + 4 g + r
    f32x4 w[STEPS];                        // id c, columns as Rows
    using Back = f32x4;
    const Back* wt;                        // [TILES][lanes], in LDS: column 16 s + c, ids 4 g + j

    __device__ void weights(const K* wr, int64_t Dp, int64_t c0) {
#pragma unroll
        for (int s = 0; s < STEPS; s++) w[s] = *reinterpret_cast<const f32x4*>(wr + lane_c() * Dp + c0 + 16 * s + 4 * lane_g());
    }
    __device__ void weights_back(const K* wc, int64_t c0, Back* to) {
        to += threadIdx.x % WAVE;
#pragma unroll
        for (int s = 0; s < TILES; s++) to[s * WAVE] = *reinterpret_cast<const Back*>(wc + (c0 + 16 * s + lane_c()) * VMAX + 4 * lane_g());
        wt = to;
    }
    static __device__ Rows rows(const E* row, int64_t c0, int64_t D) {
        Rows R;
        row += c0 + 4 * lane_g();
        over_slab(c0 + COLS <= D, [&](auto whole) {
#pragma unroll
            for (int s = 0; s < STEPS; s++) R.h[s] = whole ? pack<E, 4>::load(row + 16 * s) : get<E, 4>(row + 16 * s, D - c0 - 16 * s - 4 * lane_g());
        });
        return R;
    }
    static __device__ void clear(Rows& R) {
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int j = 0; j < 4; j++) R.h[s].v[j] = E(0.0f);
    }
    static __device__ f32x4 product(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
    __device__ f32x4 logits(const Rows& R, f32x4 l) const {
#pragma unroll
        for (int s = 0; s < STEPS; s++)
#pragma unroll
            for (int j = 0; j < 4; j++) l = product(w[s][j], float(R.h[s].v[j]), l);
        return l;
    }
    __device__ void back(const Rows& R, f32x4 dl, E* d_row, int64_t c0, int64_t D, bool store, Sums& S) const {
        const int c = lane_c(), g = lane_g();
        const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
        float one[4];                      // rows j, 4 + j, 8 + j, 12 + j of the identity
#pragma unroll
        for (int j = 0; j < 4; j++) one[j] = c == 4 * g + j ? 1.0f : 0.0f;
        f32x4 t = none;                    // id c, places 4 g + j
#pragma unroll
        for (int j = 0; j < 4; j++) t = product(dl[j], one[j], t);
        const bool whole = c0 + COLS <= D;
        d_row += c0 + 4 * g;
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            f32x4 ht = none, x = none;     // ht: column 16 s + c, places 4 g + j
            const f32x4 ws = wt[s * WAVE];
#pragma unroll
            for (int j = 0; j < 4; j++) ht = product(float(R.h[s].v[j]), one[j], ht);
#pragma unroll
            for (int j = 0; j < 4; j++) { S.dw[s] = product(ht[j], t[j], S.dw[s]); x = product(ws[j], dl[j], x); }
            if (store) {
                pack<E, 4> o;
#pragma unroll
                for (int r = 0; r < 4; r++) o.v[r] = E(x[r]);
                if (whole) o.store(d_row + 16 * s);
                else put<E, 4>(o, d_row + 16 * s, D - c0 - 16 * s - 4 * g);
            }
        }
    }
    static __device__ void begin(Sums& S) { S = {}; }
    static __device__ f32x4 end(const Sums& S, int k) { return S.dw[k]; }
    static __device__ int column(int k) { return 16 * k + 4 * lane_g(); }
};

// Place n: where its row is, and the id that it predicts (-1: it does not count)
__device__ inline void split(const Shape& S, int64_t n, int64_t& b, int64_t& t) {
    if (S.N <= UINT32_MAX) { const uint32_t m = uint32_t(n), d = uint32_t(S.T); b = m / d; t = m % d; }
    else { b = n / S.T; t = n % S.T; }
}
template <typename E> __device__ inline const E* place(const Shape& S, const E* hidden, int64_t b, int64_t t, int64_t n) {
    return hidden + (S.flat ? n * S.ht : b * S.hb + t * S.ht);
}
__device__ inline int target(const Shape& S, const void* tokens, int64_t b, int64_t t) {
    if (t + 1 >= S.T) return -1;
    const int64_t i = b * S.tb + t + 1;
    const int64_t v = S.token_bytes == 1 ? int64_t(static_cast<const uint8_t*>(tokens)[i]) : static_cast<const int64_t*>(tokens)[i];
    return v >= 0 && v < S.V && v != S.ignore ? int(v) : -1;
}

template <typename X> __device__ inline X wave_total(X x) {
#pragma unroll
    for (int d = WAVE / 2; d; d >>= 1) x += __shfl_xor(x, d, WAVE);
    return x;
}
// scale / count, from the counting workgroups' numbers
__device__ inline float mean_factor(const int64_t* counts, const float* scale) {
    int64_t k = 0;
    for (int j = threadIdx.x % WAVE; j < COUNTS; j += WAVE) k += counts[j];
    k = wave_total(k);
    return (scale ? *scale : 1.0f) / float(k > 0 ? k : 1);
}


// Logits (place c, ids 4 g + r) made the gradients of the place's loss times `w` (0 where it does not count); the loss itself
// where it is wanted (wave-uniform). The exponentials are off by some |l - top| 2^-24 of themselves, which is what the logits' own
// rounding in 32 bits moves them by.
__device__ inline float softmax(f32x4& l, int at, int V, float w, bool loss) {
    const int first = 4 * lane_g();
    const auto sum = [](float a, float b) { return a + b; };
    float top = -INFINITY, total = 0.0f, x = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; r++) if (first + r < V) top = fmaxf(top, l[r]);
    top = over_groups(top, [](float a, float b) { return fmaxf(a, b); });
    f32x4 e;
#pragma unroll
    for (int r = 0; r < 4; r++) { e[r] = first + r < V ? __expf(l[r] - top) : 0.0f; total += e[r]; }
    total = over_groups(total, sum);
    if (loss) {
        float own = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; r++) own += first + r == at ? l[r] : 0.0f;
        own = over_groups(own, sum);
        x = at >= 0 ? logf(total) + (top - own) : 0.0f;
    }
    const float up = __builtin_amdgcn_rcpf(total);
#pragma unroll
    for (int r = 0; r < 4; r++) l[r] = at >= 0 ? (e[r] * up - (first + r == at ? 1.0f : 0.0f)) * w : 0.0f;
    return x;
}

// Workgroups below `counting`: how many places count. The others: the weights, filled up with zeros to 16 ids and whole slabs,
// by ids (wr) and by columns (wc).
template <typename W, typename K>
__global__ __launch_bounds__(BLOCK) void begin_kernel(Shape S, const void* tokens, int counting, int64_t* counts, const W* weight, K* wr, K* wc) {
    if (int(blockIdx.x) < counting) {
        __shared__ int64_t lds[BLOCK / WAVE];
        int64_t k = 0;
        for (int64_t n = int64_t(blockIdx.x) * BLOCK + threadIdx.x; n < S.N; n += int64_t(COUNTS) * BLOCK) {
            int64_t b, t;
            split(S, n, b, t);
            k += target(S, tokens, b, t) >= 0;
        }
        k = wave_total(k);
        if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = k;
        __syncthreads();
        if (threadIdx.x) return;
        for (int w = 1; w < BLOCK / WAVE; w++) k += lds[w];
        counts[blockIdx.x] = k;
        return;
    }
    const int v = (blockIdx.x - counting) % VMAX;
    const int64_t i = int64_t((blockIdx.x - counting) / VMAX) * BLOCK + threadIdx.x;
    if (i >= S.Dp) return;
    const K x = v < S.V && i < S.D ? K(float(weight[v * S.D + i])) : K(0.0f);
    wr[v * S.Dp + i] = x;
    if (wc) wc[i * VMAX + v] = x;
}

// Logits, losses and, with GRADS, all gradients in one pass over hidden; a wave for each slab of the row
template <typename M, bool GRADS>
__global__ __launch_bounds__(MOST_WAVES* WAVE)
void fused_kernel(Shape S, const typename M::E* __restrict__ hidden, const void* __restrict__ tokens, const typename M::K* __restrict__ wr,
                  const typename M::K* __restrict__ wc, const int64_t* counts, const float* scale, const float* __restrict__ factor, float* __restrict__ each,
                  typename M::E* __restrict__ d_hidden, double* sums, float* __restrict__ parts) {
    extern __shared__ f32x4 lds[];         // partial logits, for this tile and the one before: [2][waves][lanes]; then the waves' wt
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), waves = blockDim.x / WAVE, lane = threadIdx.x % WAVE, c = lane_c();
    const int64_t c0 = int64_t(wave) * M::COLS;
    struct Next { typename M::Rows rows; int at; float w; } next;
    auto fetch = [&](int64_t tile) {
        const int64_t n = tile * TILE + c;
        const bool on = n < S.N;
        int64_t b, t;
        split(S, on ? n : 0, b, t);
        next.rows = M::rows(place(S, hidden, b, t, on ? n : 0), c0, S.D);
        next.at = on ? target(S, tokens, b, t) : -1;
        if (GRADS) next.w = factor && on ? factor[n] : 0.0f;
    };
    const int64_t tiles = (S.N + TILE - 1) / TILE;
    if (blockIdx.x < tiles) fetch(blockIdx.x);
    M m;
    m.weights(wr, S.Dp, c0);
    if (GRADS) m.weights_back(wc, c0, reinterpret_cast<typename M::Back*>(lds + 2 * waves * WAVE) + wave * M::TILES * WAVE);
    typename M::Sums sum;
    M::begin(sum);
    const float base = GRADS && counts ? mean_factor(counts, scale) : 0.0f;
    double loss = 0.0;
    int turn = 0;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= 1) {
        Next now = next;
        if (tile + gridDim.x < tiles) fetch(tile + gridDim.x);
        if (GRADS && now.at < 0) M::clear(now.rows);
        f32x4 l = m.logits(now.rows, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        if (waves > 1) {
            f32x4* mine = lds + turn * waves * WAVE;
            mine[wave * WAVE + lane] = l;
            __syncthreads();               // (the other half is free again: every wave has passed the tile before)
            if (!GRADS && wave) continue;
            mine += lane;
            l = mine[0];
            int k = 1;
            for (; !GRADS && k + 3 < waves; k += 4) {      // (four reads under way at a time; with gradients there are no registers for them)
                const f32x4 a = mine[k * WAVE], b = mine[(k + 1) * WAVE], d = mine[(k + 2) * WAVE], e = mine[(k + 3) * WAVE];
                l += (a + b) + (d + e);
            }
            for (; k < waves; k++) l += mine[k * WAVE];
        }
        const float x = softmax(l, now.at, S.V, factor ? now.w : base, wave == 0);
        const int64_t n = tile * TILE + c;
        if (wave == 0 && lane < TILE && n < S.N) {
            loss += double(x);
            if (each) each[n] = x;
        }
        if (GRADS) m.back(now.rows, l, d_hidden + n * S.D, c0, S.D, n < S.N, sum);
    }
    if (wave == 0) {
        loss = wave_total(loss);
        if (lane == 0) sums[blockIdx.x] = loss;
    }
    if (GRADS && c < S.V) {
#pragma unroll
        for (int k = 0; k < M::TILES; k++) *reinterpret_cast<f32x4*>(parts + (int64_t(blockIdx.x) * S.V + c) * S.Dp + c0 + M::column(k)) = M::end(sum, k);
    }
}

// Logits and losses of a tile by one wave, over all columns; with d_logits, their gradients ([N, 16])
template <typename M>
__global__ __launch_bounds__(BLOCK) void place_kernel(Shape S, const typename M::E* __restrict__ hidden, const void* __restrict__ tokens,
                                                      const typename M::K* __restrict__ wr, const int64_t* counts, const float* scale,
                                                      const float* __restrict__ factor, float* __restrict__ each, f32x4* __restrict__ d_logits, double* sums) {
    __shared__ double lds[BLOCK / WAVE];
    const int lane = threadIdx.x % WAVE, c = lane_c();
    const float base = d_logits && counts ? mean_factor(counts, scale) : 0.0f;
    double loss = 0.0;
    const int64_t tiles = (S.N + TILE - 1) / TILE;
    for (int64_t tile = int64_t(blockIdx.x) * (BLOCK / WAVE) + threadIdx.x / WAVE; tile < tiles; tile += int64_t(gridDim.x) * (BLOCK / WAVE)) {
        const int64_t n = tile * TILE + c;
        const bool on = n < S.N;
        int64_t b, t;
        split(S, on ? n : 0, b, t);
        const typename M::E* row = place(S, hidden, b, t, on ? n : 0);
        const int at = on ? target(S, tokens, b, t) : -1;
        f32x4 l = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t c0 = 0; c0 < S.D; c0 += M::COLS) {
            M m;
            m.weights(wr, S.Dp, c0);
            l = m.logits(M::rows(row, c0, S.D), l);
        }
        const float x = softmax(l, at, S.V, factor && on ? factor[n] : base, true);
        if (lane < TILE && on) {
            loss += double(x);
            if (each) each[n] = x;
        }
        if (d_logits && on) d_logits[n * 4 + lane_g()] = l;
    }
    loss = wave_total(loss);
    if (lane == 0) lds[threadIdx.x / WAVE] = loss;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < BLOCK / WAVE; w++) loss += lds[w];
    sums[blockIdx.x] = loss;
}

// d_hidden and d_weight from d_logits, a wave for each slab
template <typename M>
__global__ __launch_bounds__(BLOCK) void grad_kernel(Shape S, const typename M::E* __restrict__ hidden, const void* __restrict__ tokens,
                                                     const typename M::K* __restrict__ wc, const f32x4* __restrict__ d_logits,
                                                     typename M::E* __restrict__ d_hidden, float* __restrict__ parts) {
    const int c = lane_c();
    const int64_t c0 = (int64_t(blockIdx.x) * (BLOCK / WAVE) + threadIdx.x / WAVE) * M::COLS;
    if (c0 >= S.Dp) return;
    M m;
    __shared__ typename M::Back room[BLOCK / WAVE][M::TILES * WAVE];
    m.weights_back(wc, c0, room[threadIdx.x / WAVE]);
    typename M::Sums sum;
    M::begin(sum);
    const int64_t tiles = (S.N + TILE - 1) / TILE;
    for (int64_t tile = blockIdx.y; tile < tiles; tile += gridDim.y) {
        const int64_t n = tile * TILE + c;
        const bool on = n < S.N;
        int64_t b, t;
        split(S, on ? n : 0, b, t);
        typename M::Rows rows = M::rows(place(S, hidden, b, t, on ? n : 0), c0, S.D);
        const f32x4 dl = on ? d_logits[n * 4 + lane_g()] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!on || target(S, tokens, b, t) < 0) M::clear(rows);
        m.back(rows, dl, d_hidden + n * S.D, c0, S.D, on, sum);
    }
    if (c < S.V) {
#pragma unroll
        for (int k = 0; k < M::TILES; k++) *reinterpret_cast<f32x4*>(parts + (int64_t(blockIdx.y) * S.V + c) * S.Dp + c0 + M::column(k)) = M::end(sum, k);
    }
}

// The mean loss (the last workgroup), and d_weight from the workgroups' parts: 64 columns a workgroup, a run of parts a wave
template <typename W>
__global__ __launch_bounds__(END_WAVES* WAVE) void end_kernel(Shape S, const int64_t* counts, const double* sums, int nsums, float* loss, const float* __restrict__ parts,
                                                              int nparts, W* __restrict__ d_weight) {
    __shared__ float lds[END_WAVES][WAVE];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    if (loss && blockIdx.x == gridDim.x - 1) {
        if (wave) return;
        int64_t k = 0;
        for (int j = lane; j < COUNTS; j += WAVE) k += counts[j];
        k = wave_total(k);
        double s = 0.0;
        for (int j = lane; j < nsums; j += WAVE) s += sums[j];
        s = wave_total(s);
        if (lane == 0) *loss = float(s / double(k > 0 ? k : 1));
        return;
    }
    const int64_t e = int64_t(blockIdx.x) * WAVE + lane, size = S.V * S.Dp;
    float x = 0.0f;
    if (e < size) {
#pragma unroll 8
        for (int p = wave; p < nparts; p += END_WAVES) x += parts[p * size + e];
    }
    lds[wave][lane] = x;
    __syncthreads();
    if (wave || e >= size) return;
#pragma unroll
    for (int w = 1; w < END_WAVES; w++) x += lds[w][lane];
    const int64_t v = e / S.Dp, i = e % S.Dp;
    if (i < S.D) d_weight[v * S.D + i] = W(x);
}

// How a call is cut up: D in whole slabs, waves of a fused workgroup (0: the row has more slabs than that), workgroups
struct Cut { int64_t Dp; int waves, groups; };
Cut cut_of(int64_t N, int64_t D, bool narrow, bool gradients) {
    const int64_t cols = narrow ? 128 : 64, slabs = (D + cols - 1) / cols, tiles = (N + TILE - 1) / TILE;
    Cut k;
    k.Dp = slabs * cols;
    k.waves = slabs <= MOST_WAVES ? int(slabs) : 0;
    const int64_t most = k.waves ? 256 * ((gradients ? 16 : 24) / k.waves) : 256;      // of 256 CUs, 16 or 24 waves a CU
    const int64_t rounds = (tiles + most - 1) / most;                          // all workgroups have as many tiles, one less here and there
    int64_t groups = (tiles + rounds - 1) / rounds;
    // With gradients and several workgroups a CU: as many on each CU (5 x 2,049 x 500 float32 as 321 workgroups 24.5 us, as 512
    // 20.3; 33,600 x 512 57.7 and 53.5). With one a CU or without gradients more would cost: 25,000 x 1,000 float32 as 224
    // 76.2 us, as 256 77.8; losses of 131,072 x 128 bfloat16 34 and 42.
    if (gradients && most > 256) groups = std::min({(groups + 255) / 256 * 256, most, tiles});
    k.groups = int(groups);
    return k;
}
constexpr int PLACE_GROUPS = 2048;

struct Work { int64_t* counts; double* sums; char *wr, *wc; float *d_logits, *parts; uint64_t bytes; };
Work layout(void* work, int64_t N, int64_t D, int32_t V, bool narrow, bool gradients) {
    const Cut k = cut_of(N, D, narrow, gradients);
    const uint64_t e = narrow ? 2 : 4;
    char* at = static_cast<char*>(work);
    auto take = [&](uint64_t bytes) { char* p = at; at += (bytes + 15) & ~15ull; return p; };
    Work w;
    w.counts = reinterpret_cast<int64_t*>(take(COUNTS * 8));
    w.sums = reinterpret_cast<double*>(take((k.groups > PLACE_GROUPS ? k.groups : PLACE_GROUPS) * 8));
    w.wr = take(VMAX * k.Dp * e);
    w.wc = gradients ? take(VMAX * k.Dp * e) : nullptr;
    w.d_logits = reinterpret_cast<float*>(gradients && !k.waves ? take(uint64_t(N) * VMAX * 4) : nullptr);
    w.parts = reinterpret_cast<float*>(gradients ? take(uint64_t(k.groups) * V * k.Dp * 4) : nullptr);
    w.bytes = uint64_t(at - static_cast<char*>(work));
    return w;
}

template <typename M, typename W>
int32_t run(Shape S, const void* hidden_, const void* weight, const void* tokens, const float* scale, const float* factor, float* each, float* loss, void* d_hidden_,
            void* d_weight, void* work, hipStream_t st, char* err, size_t errcap) {
    using E = typename M::E;
    using K = typename M::K;
    const bool narrow = sizeof(K) == 2, grads = d_hidden_;
    const Work w = layout(work, S.N, S.D, S.V, narrow, grads);
    const Cut k = cut_of(S.N, S.D, narrow, grads);
    S.Dp = k.Dp;
    const E* hidden = static_cast<const E*>(hidden_);
    E* d_hidden = static_cast<E*>(d_hidden_);
    K *wr = reinterpret_cast<K*>(w.wr), *wc = reinterpret_cast<K*>(w.wc);
    const bool mean = loss || (grads && !factor);
    const int counting = mean ? COUNTS : 0;
    begin_kernel<W, K><<<counting + VMAX * ((k.Dp + BLOCK - 1) / BLOCK), BLOCK, 0, st>>>(S, tokens, counting, w.counts, static_cast<const W*>(weight), wr, wc);
    const int64_t* counts = mean ? w.counts : nullptr;
    int nsums = k.groups;
    const size_t exchange = 2 * k.waves * WAVE * sizeof(f32x4);
    if (grads && k.waves) {
        fused_kernel<M, true><<<k.groups, k.waves * WAVE, exchange + k.waves * M::TILES * WAVE * sizeof(typename M::Back), st>>>(S, hidden, tokens, wr, wc, counts, scale, factor, each, d_hidden, w.sums, w.parts);
    } else if (k.waves) {
        fused_kernel<M, false><<<k.groups, k.waves * WAVE, exchange, st>>>(S, hidden, tokens, wr, nullptr, nullptr, nullptr, nullptr, each, nullptr, w.sums, nullptr);
    } else {
        const int64_t need = (S.N + TILE * (BLOCK / WAVE) - 1) / (TILE * (BLOCK / WAVE));
        nsums = int(need < PLACE_GROUPS ? need : PLACE_GROUPS);
        place_kernel<M><<<nsums, BLOCK, 0, st>>>(S, hidden, tokens, wr, counts, scale, factor, each, reinterpret_cast<f32x4*>(w.d_logits), w.sums);
        if (grads)
            grad_kernel<M><<<dim3((k.Dp + M::COLS * (BLOCK / WAVE) - 1) / (M::COLS * (BLOCK / WAVE)), k.groups), BLOCK, 0, st>>>(
                S, hidden, tokens, wc, reinterpret_cast<const f32x4*>(w.d_logits), d_hidden, w.parts);
    }
    if (loss || grads)
        end_kernel<W><<<(grads ? (S.V * k.Dp + WAVE - 1) / WAVE : 0) + (loss ? 1 : 0), END_WAVES * WAVE, 0, st>>>(S, w.counts, w.sums, nsums, loss, w.parts, k.groups,
                                                                                                              static_cast<W*>(d_weight));
    return launched(err, errcap);
}

}  // namespace

extern "C" {

uint64_t pv_next_base_loss_work_bytes(int64_t B, int64_t T, int64_t D, int32_t V, int32_t gradients) {
    if (B <= 0 || T <= 0 || D <= 0 || V <= 0 || B > (int64_t(1) << 40) / T) return 0;
    const uint64_t a = layout(nullptr, B * T, D, V, true, gradients).bytes, b = layout(nullptr, B * T, D, V, false, gradients).bytes;
    return a > b ? a : b;
}

int32_t pv_next_base_loss_hip(const void* hidden, const void* weight, const void* tokens, int64_t B, int64_t T, int64_t D, int32_t V, int64_t hidden_b,
                              int64_t hidden_t, int64_t tokens_b, int64_t ignore, int32_t dtype, int32_t weight_dtype, int32_t token_bytes, const float* scale,
                              const float* factor, float* each, float* loss, void* d_hidden, void* d_weight, void* work, uint64_t work_bytes, void* stream,
                              char* err, size_t errcap) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, errcap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (weight_dtype != dtype && weight_dtype != PV_F32) return fail(PV_EARG, err, errcap, "weight_dtype: hidden's, or PV_F32");
    if (token_bytes != 1 && token_bytes != 8) return fail(PV_EARG, err, errcap, "token_bytes: 1 or 8");
    if (B < 1 || T < 1 || D < 1 || D > MOST_COLUMNS || B > (int64_t(1) << 40) / T) return fail(PV_EARG, err, errcap, "shape: B, T, D >= 1, D <= 2^23, B * T <= 2^40");
    if (V < 1 || V > VMAX) return fail(PV_EARG, err, errcap, "V: 1 to 16 ids");
    if (!hidden || !weight || !tokens || !d_hidden != !d_weight) return fail(PV_EARG, err, errcap, "null argument");
    if (!work || work_bytes < pv_next_base_loss_work_bytes(B, T, D, V, d_hidden != nullptr) || !aligned(work, 16))
        return fail(PV_EARG, err, errcap, "work: too small, or not 16-byte aligned");
    Shape S{B, T, D, B * T, hidden_b, hidden_t, tokens_b, ignore, 0, V, token_bytes, B == 1 || hidden_b == T * hidden_t};
    const bool narrow = dtype != PV_F32 && weight_dtype == dtype;
    const hipStream_t st = hipStream_t(stream);
    if (narrow && dtype == PV_BF16) return run<H2<bf16>, bf16>(S, hidden, weight, tokens, scale, factor, each, loss, d_hidden, d_weight, work, st, err, errcap);
    if (narrow) return run<H2<f16>, f16>(S, hidden, weight, tokens, scale, factor, each, loss, d_hidden, d_weight, work, st, err, errcap);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        return run<F3<E>, float>(S, hidden, weight, tokens, scale, factor, each, loss, d_hidden, d_weight, work, st, err, errcap);
    });
}

}  // extern "C"
