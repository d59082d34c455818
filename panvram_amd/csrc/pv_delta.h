// What the kernels of the gated delta rule (pv_delta.hip, pv_delta_back.hip) share: matrix operands and their tiles in LDS, the
// records that one kernel leaves another, and the sizes of a call.
//
// Operands. A product of 16 x 16 x 32 has, in lane l = 16 g + m, of its left operand row m and of its right one column m, at eight
// places of the 32 that are summed over; and of its result column m, rows 4 g .. 4 g + 3. Which eight places a lane has is free as
// long as both operands agree: here they are 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3 of each 32. So two results, rows 0..15 and
// 16..31 of some matrix, are an operand of the next product as they are, with their rows summed over: a state and all that is made
// from it stay in registers.
//
// Held as. Of tensors in 16 bits the operands are float16, scaled by powers of two: keys and queries step by step, to lengths near 64,
// and what is computed in 32 bits column by column of the state, so that the column's largest value is 2^13 or a little more and what
// falls below float16's numbers is 2^-37 of that. A product's scale is a number of the lane, as a lane has one column. `wide` operands
// are two float16, a value and what its rounding left: 22 bits. `narrow` ones are the first alone, 11 bits, which only outputs in
// 16 bits are made from. Wide are the states and all that they are made from: they are kept and returned in 32 bits. (Two bfloat16 in
// their place, without any scale, left states off by 4e-6 and outputs in bfloat16 by 1.7 times their own rounding.) Of tensors in
// float32 the operands are float32, eight products of 16 x 16 x 4 in the place of one of 32, and scales are 1.
#pragma once
#include "pv_ops.h"

#include <type_traits>

namespace pvd {

using namespace pvo;

constexpr int C = 64;                      // steps of a chunk
constexpr int MAX_K = 128;

using f4 = __attribute__((ext_vector_type(4))) float;
using h8 = __attribute__((ext_vector_type(8))) _Float16;

// What operands are held as for tensors of E: S, how many of them a wide one takes; lengths of keys and queries, and the scale
// of the matrices of 64 x 64, whose elements are 1 at most
template <typename E> struct Rep { using S = f16; };
template <> struct Rep<float> { using S = float; };
template <typename S> constexpr int wide_of = sizeof(S) == 2 ? 2 : 1;
template <typename S> constexpr float LONG = sizeof(S) == 2 ? 64.0f : 1.0f;
template <typename S> constexpr float SQUARE = sizeof(S) == 2 ? 4096.0f : 1.0f;

// The power of two for a column whose largest value is `most`, and one over it (of numbers below 2^-113 the largest there is)
struct Scale { float up, down; };
template <typename S> __device__ inline Scale scale_of(float most) {
    if constexpr (sizeof(S) == 4) return {1.0f, 1.0f};
    uint32_t e = __float_as_uint(most) >> 23;
    e = e < 14 ? 14 : e;
    return {__uint_as_float((267 - e) << 23), __uint_as_float((e - 13) << 23)};
}
// Of a step whose length is 1 / r: what its elements are multiplied by, and what is left of r
template <typename S> __device__ inline float length_up(float r) {
    if constexpr (sizeof(S) == 4) return r == 0.0f ? 0.0f : 1.0f;
    return __uint_as_float(__float_as_uint(r) & 0x7f800000u) * LONG<S>;
}
template <typename S> __device__ inline float length_rest(float r) {
    if constexpr (sizeof(S) == 4) return r;
    return r == 0.0f ? 0.0f : __uint_as_float((__float_as_uint(r) & 0x7fffffu) | 0x3f800000u) * (1.0f / LONG<S>);
}

// The largest over the four lanes that have a column
__device__ inline float over_column(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
template <int N> __device__ inline float largest(const f4 (&v)[N]) {
    float x = 0.0f;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) x = fmaxf(x, fabsf(v[n][r]));
    return x;
}

template <typename S, int PARTS> struct Frag;
template <int PARTS> struct Frag<f16, PARTS> { h8 p[PARTS]; };
template <int PARTS> struct Frag<float, PARTS> { float v[8]; };

template <int A, int B> __device__ inline void mma(f4& acc, const Frag<f16, A>& a, const Frag<f16, B>& b) {
#pragma unroll
    for (int i = A - 1; i >= 0; i--)
#pragma unroll
        for (int j = B - 1; j >= 0; j--)
            if (i + j < (A > B ? A : B)) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.p[i], b.p[j], acc, 0, 0, 0);   // (not rest times rest)
}
template <int A, int B> __device__ inline void mma(f4& acc, const Frag<float, A>& a, const Frag<float, B>& b) {
#pragma unroll
    for (int j = 0; j < 8; j++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], acc, 0, 0, 0);
}

// Two results, rows 0..15 and 16..31, times `up` as an operand summed over their rows
template <typename S, int PARTS> __device__ inline Frag<S, PARTS> frag_of(const f4& lo, const f4& hi, float up) {
    Frag<S, PARTS> f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float x = j < 4 ? lo[j] : hi[j - 4];
        if constexpr (sizeof(S) == 4) {
            f.v[j] = x;
        } else {
            const f16 h = f16(x * up);
            f.p[0][j] = h;
            if constexpr (PARTS == 2) f.p[1][j] = f16(fmaf(x, up, -float(h)));
        }
    }
    return f;
}
template <int PARTS> __device__ inline const Frag<float, 1>& narrow(const Frag<float, PARTS>& f) { return f; }
template <int PARTS> __device__ inline Frag<f16, 1> narrow(const Frag<f16, PARTS>& f) { return {{f.p[0]}}; }

// Where column c of a row lies in a tile: of each 32 the places of a lane are neighbours
__host__ __device__ constexpr int place(int c) { return (c & ~31) | (c & 12) << 1 | (c & 16) >> 2 | (c & 3); }

// A tile in LDS: rows of COLS elements, of PARTS parts each in a plane of its own. The padding spreads rows over banks.
template <typename S_, int ROWS, int COLS, int PARTS = 1> struct Tile {
    using S = S_;
    static constexpr int ROW = COLS + 16 / sizeof(S), PLANE = ROWS * ROW, SIZE = PLANE * PARTS;
    S* p;
    // rows r0 .. r0 + 15, summed over columns 32 kb ..
    __device__ Frag<S, PARTS> rows(int r0, int kb) const {
        const int l = threadIdx.x % WAVE;
        const S* at = p + (r0 + l % 16) * ROW + kb * 32 + (l / 16) * 8;
        Frag<S, PARTS> f;
        if constexpr (sizeof(S) == 2) {
#pragma unroll
            for (int k = 0; k < PARTS; k++) f.p[k] = *reinterpret_cast<const h8*>(at + k * PLANE);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) f.v[j] = at[j];
        }
        return f;
    }
    // the same of its first part alone
    __device__ Frag<S, 1> rows_narrow(int r0, int kb) const { return Tile<S, ROWS, COLS, 1>{p}.rows(r0, kb); }
    // columns c0 .. c0 + 15, summed over rows 32 kb ..
    __device__ Frag<S, PARTS> cols(int c0, int kb) const {
        const int l = threadIdx.x % WAVE, g = l / 16, m = l % 16;
        Frag<S, PARTS> f;
        if constexpr (sizeof(S) == 2) {    // (a transposing read: 16 lanes give 4 rows of 4 neighbours each, and take 4 rows of a column each)
            using quad = __attribute__((ext_vector_type(4))) short;
            const S* at = p + (kb * 32 + g * 4 + m / 4) * ROW + place(c0 + 4 * (m % 4));
#pragma unroll
            for (int k = 0; k < PARTS; k++) {
                union { quad q[2]; h8 h; } u;
#pragma unroll
                for (int h = 0; h < 2; h++)
                    u.q[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) quad*)(at + k * PLANE + 16 * h * ROW));
                f.p[k] = u.h;
            }
        } else {
            const S* at = p + (kb * 32 + g * 4) * ROW + place(c0 + m);
#pragma unroll
            for (int j = 0; j < 8; j++) f.v[j] = at[(j % 4 + j / 4 * 16) * ROW];
        }
        return f;
    }
    __device__ Frag<S, 1> cols_narrow(int c0, int kb) const { return Tile<S, ROWS, COLS, 1>{p}.cols(c0, kb); }
    // eight neighbouring places of a row, in the first part
    __device__ void put_places(int row, int at, const pack<S, 8>& v) const { v.store(p + row * ROW + at); }
    __device__ S get(int row, int c) const { return p[row * ROW + place(c)]; }
    // eight neighbouring columns of a row, c a multiple of 8
    __device__ void put(int row, int c, const S (&v)[8]) const {
        S* at = p + row * ROW + place(c);
        using quad = pack<S, 4>;
        quad a, b;
#pragma unroll
        for (int j = 0; j < 4; j++) { a.v[j] = v[j]; b.v[j] = v[4 + j]; }
        a.store(at);
        b.store(at + 8);                   // (place(c + 4))
    }
};

// Rows of queries or keys on their way from memory to a tile of 64 x DK, eight elements a lane. No load depends on a branch that
// lanes take differently, as it would be waited for there: steps past the last are read as the last one (they have length 0, and
// their elements come out as 0), elements past a row's end are not read, and its last eight are read as they lie, where K is no
// multiple of 8, and put one by one.
template <typename E, int DK, int THREADS> struct Rows {
    using S = typename Rep<E>::S;
    static constexpr int PER = DK / 8, COUNT = C * PER / THREADS;
    pack<E, 8> v[COUNT];
    static __device__ int column(int K) {                  // of the lane's first element
        const int c = threadIdx.x % PER * 8;
        return c + 8 <= K ? c : K >= 8 ? K - 8 : 0;
    }
    static __device__ int row(int j) { return (threadIdx.x + j * THREADS) / PER; }
    __device__ void load(const E* at, int64_t stride, int rows, int K) {
        const int c = column(K);
        if (K >= 8) {
#pragma unroll
            for (int j = 0; j < COUNT; j++) v[j] = pack<E, 8>::load(at + (row(j) < rows ? row(j) : rows - 1) * stride + c);
        } else {
#pragma unroll
            for (int j = 0; j < COUNT; j++) v[j] = pack<E, 8>::load_part(at + (row(j) < rows ? row(j) : rows - 1) * stride, K);
        }
    }
    __device__ float square(int j, int K) const {          // of the lane's own elements, none of them a neighbour's too
        const int own = K - int(threadIdx.x % PER * 8);
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float x = float(v[j].v[e]);
            const bool on = K < 8 ? own > 0 : own >= 8 || 8 - e <= own;
            s = on ? fmaf(x, x, s) : s;
        }
        return s;
    }
    template <typename T> __device__ void put(const T& tile, int j, float up, int K) const {
        if (int(threadIdx.x % PER * 8) >= K) return;
        S x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = S(float(v[j].v[e]) * up);
        const int c = column(K);
        if (c % 8 == 0) tile.put(row(j), c, x);
        else
#pragma unroll
            for (int e = 0; e < 8; e++) tile.p[row(j) * T::ROW + place(c + e)] = x[e];
    }
    // the columns behind the last, once
    template <typename T> static __device__ void clear(const T& tile, int K) {
        if (K == DK) return;
        const S zero[8] = {};
        for (int p = threadIdx.x; p < C * PER; p += THREADS) tile.put(p / PER, p % PER * 8, zero);
        __syncthreads();
    }
};

// The call: B sequences of T steps, H query and key heads of K, G value heads of V. Strides in elements.
struct Shape {
    int64_t B, T;
    int32_t H, G, K, V;
    int64_t qb, qt, qh, kb, kt, kh, vb, vt, vh;            // query, key, value: of a sequence, a step, a head
    int64_t ab, at, ag, wb, wt, wg;                        // gate, write: of a sequence, a step, a head
    int64_t ob, ot, og;                                    // d_out
    int64_t chunks;                                        // of T
    int32_t vp;                                            // V up to a multiple of 16
    float eps;
};

// What is known of a chunk's steps before its state is: one record for each chunk of each value head.
//   x     g r: g what a step keeps of the state before the chunk (0 past a reset), r what is left of one over the key's length
//   b     sigmoid(write)
//   l     l r: l what is left of a step's addition at the chunk's end
//   q     g r of the query
//   end   what the chunk keeps of the state;  cut: a bit for each step that drops the state before it
struct Steps {
    float x[C], b[C], l[C], q[C], rk[C], rq[C], hi[C], lo[C];      // hi + lo: the logarithm of what is kept, summed up from the chunk's first step
    float end;
    uint32_t cut[2], unused;
};
template <typename S> struct Chunk {
    S inv[wide_of<S>][C][C], pair[wide_of<S>][C][C];       // (I + A)^-1 and M q k^T, times SQUARE, columns at their places
    Steps steps;
};

// Steps that a record's cut lets through: whether step j's addition is still there at step i >= j
__device__ inline int since(uint64_t cut, int i) {         // the last step up to i that drops the state, or -1
    const uint64_t m = cut & (~0ull >> (63 - i));
    return m ? 63 - __builtin_clzll(m) : -1;
}

// What the forward pass keeps for the backward pass, and what the walk backwards leaves for the gradients: arrays of the same
// shapes, for a chunk of a value head. By columns of the state or of values, vp of them:
//   states   [vp][DK]: S before the chunk, or the gradient of S after it; rows at their places
//   steps    [vp][64]: U, or the gradient of b D; steps at their places
//   scales   [3][vp]: what the columns of states, of steps, and (backwards) of the gradient of out are to be multiplied by
template <typename S> struct Kept {
    S *states, *steps;
    float* scales;
    Kept(void* p, const Shape& s, int dk) : states(static_cast<S*>(p)), steps(states + s.B * s.G * s.chunks * int64_t(s.vp) * dk),
                                            scales(reinterpret_cast<float*>(steps + s.B * s.G * s.chunks * int64_t(s.vp) * C)) {}
};
// An operand's first part, eight places of a column, to memory
template <typename S, int PARTS> __device__ inline void leave(S* to, const Frag<S, PARTS>& f) {
    pack<S, 8> o;
    __builtin_memcpy(&o, &f, sizeof o);
    o.store(to);
}
inline uint64_t kept_bytes(uint64_t rows, int32_t dk, int32_t dtype) { return rows * (uint64_t(dk + C) * (dtype == PV_F32 ? 4 : 2) + 12); }

// A chunk's steps on their way from memory to LDS
template <int THREADS> struct StepsOnTheirWay {
    static constexpr int N = int(sizeof(Steps) / 4), COUNT = (N + THREADS - 1) / THREADS;
    float v[COUNT];
    __device__ void load(const Steps& s) {
        const float* from = reinterpret_cast<const float*>(&s);
#pragma unroll
        for (int j = 0; j < COUNT; j++) {
            const int at = threadIdx.x + j * THREADS;
            v[j] = from[at < N ? at : N - 1];
        }
    }
    __device__ void put(Steps& s) const {
        float* to = reinterpret_cast<float*>(&s);
#pragma unroll
        for (int j = 0; j < COUNT; j++) if (int(threadIdx.x) + j * THREADS < N) to[threadIdx.x + j * THREADS] = v[j];
    }
};
// A matrix of 64 x 64 from a record, in PARTS parts, on its way
template <typename S, int PARTS, int THREADS> struct SquareOnItsWay {
    static constexpr int P = 16 / sizeof(S), COUNT = C * C / P / THREADS;
    pack<S, P> v[PARTS][COUNT];
    __device__ void load(const S (*from)[C][C]) {
#pragma unroll
        for (int w = 0; w < PARTS; w++)
#pragma unroll
            for (int j = 0; j < COUNT; j++) v[w][j] = pack<S, P>::load(&from[w][0][0] + (threadIdx.x + j * THREADS) * P);
    }
    template <typename T> __device__ void put(const T& tile) const {
#pragma unroll
        for (int w = 0; w < PARTS; w++)
#pragma unroll
            for (int j = 0; j < COUNT; j++) {
                const int at = (threadIdx.x + j * THREADS) * P;
                v[w][j].store(tile.p + w * T::PLANE + at / C * T::ROW + at % C);
            }
    }
};
// A lane's sixteen elements of a column of values: rows 16 it + 4 g + r. Steps past the last are the last one's.
template <typename E> struct Sixteen {
    E v[16];
    __device__ void load(const E* at, int64_t stride, int rows) {
        const int g = threadIdx.x % WAVE / 16;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int i = 16 * (j / 4) + 4 * g + j % 4;
            v[j] = at[(i < rows ? i : rows - 1) * stride];
        }
    }
    __device__ f4 four(int it, bool on) const {
        f4 x;
#pragma unroll
        for (int r = 0; r < 4; r++) x[r] = on ? float(v[4 * it + r]) : 0.0f;
        return x;
    }
};

// The value heads that share a query and key head are neighbours
__device__ inline int shared(const Shape& S, int g) { return g / (S.G / S.H); }

// f of a number of key columns that kernels are made for, K or more
template <typename F> int32_t with_k(int32_t K, F&& f) {
    if (K <= 32) return f(std::integral_constant<int, 32>{});
    if (K <= 64) return f(std::integral_constant<int, 64>{});
    return f(std::integral_constant<int, 128>{});
}


// The call's sizes and strides: of query, key, value, gate and write in their order, each of a sequence, a step and a head
inline int32_t shape_of(int64_t B, int64_t T, int32_t H, int32_t G, int32_t K, int32_t V, const int64_t* strides, float eps, int32_t dtype, Shape& S, char* err,
                        size_t cap) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, cap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (B < 1 || T < 1 || H < 1 || G < H || G % H || V < 1 || V > 1 << 16)
        return fail(PV_EARG, err, cap, "shape: B, T, H >= 1, G a multiple of H, 1 <= V <= 65,536");
    if (K < 1 || K > MAX_K) return fail(PV_EARG, err, cap, "shape: 1 <= K <= 128");
    const int64_t chunks = (T + C - 1) / C, heads = B * G;
    // a launch's work items: four waves for a chunk, or for 32 columns of a state
    if (B >= int64_t(1) << 24 || G >= 1 << 24 || T >= int64_t(1) << 31 || heads >= int64_t(1) << 24 || heads * chunks >= int64_t(1) << 24 ||
        heads * ((V + 31) / 32) >= int64_t(1) << 24)
        return fail(PV_EARG, err, cap, "too many chunks of 64 steps, or columns of states: fewer than 2^24");
    if (!strides) return fail(PV_EARG, err, cap, "null argument");
    for (int i = 1; i < 15; i += 3) if (strides[i] < -(1 << 24) || strides[i] > 1 << 24) return fail(PV_EARG, err, cap, "stride: a step's is 2^24 elements at most");
    S = {B, T, H, G, K, V, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7], strides[8], strides[9], strides[10], strides[11],
         strides[12], strides[13], strides[14], 0, 0, 0, chunks, (V + 15) / 16 * 16, eps};
    return PV_OK;
}

}  // namespace pvd
