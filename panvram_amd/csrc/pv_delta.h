// What the kernels of the gated delta rule (pv_delta.hip, pv_delta_back.hip) share: matrix operands and their tiles in LDS, the
// records that one kernel leaves another, and the sizes of a call.
//
// Operands. A product of 16 x 16 x 32 has, in lane l = 16 g + m, of its left operand row m and of its right one column m, at eight
// places of the 32 that are summed over; and of its result column m, rows 4 g .. 4 g + 3. Which eight places a lane has is free as
// long as both operands agree: here they are 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3 of each 32. So two results, rows 0..15 and
// 16..31 of some matrix, are an operand of the next product as they are, with their rows summed over: a state and all that is made
// from it stay in registers.
//
// Held as. Of bfloat16 tensors the operands that come from memory are one bfloat16 each. What is computed in 32 bits goes into
// another product either as two of them, a value and what its rounding left (`wide`: 16 bits, off by 2^-17 of itself), or as one
// (`narrow`, 2^-9). Wide are the states and all that they are made from, since the states are kept and returned in 32 bits; narrow is
// what only reaches outputs of bfloat16. float16 and float32 are products of float32, eight of 16 x 16 x 4 in the place of one of 32.
#pragma once
#include "pv_ops.h"

#include <type_traits>

namespace pvd {

using namespace pvo;

constexpr int C = 64;                      // steps of a chunk
constexpr int MAX_K = 128;

using f4 = __attribute__((ext_vector_type(4))) float;
using h8 = __attribute__((ext_vector_type(8))) __bf16;
using h4 = __attribute__((ext_vector_type(4))) __bf16;

// What operands are held as for tensors of E: S, and how many of them a wide one takes
template <typename E> struct Rep { using S = float; static constexpr int WIDE = 1; };
template <> struct Rep<bf16> { using S = bf16; static constexpr int WIDE = 2; };

template <typename S, int PARTS> struct Frag;
template <int PARTS> struct Frag<bf16, PARTS> { h8 p[PARTS]; };
template <int PARTS> struct Frag<float, PARTS> { float v[8]; };

template <int A, int B> __device__ inline void mma(f4& acc, const Frag<bf16, A>& a, const Frag<bf16, B>& b) {
#pragma unroll
    for (int i = A - 1; i >= 0; i--)
#pragma unroll
        for (int j = B - 1; j >= 0; j--)
            if (i + j < (A > B ? A : B)) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], acc, 0, 0, 0);   // (not rest times rest)
}
template <int A, int B> __device__ inline void mma(f4& acc, const Frag<float, A>& a, const Frag<float, B>& b) {
#pragma unroll
    for (int j = 0; j < 8; j++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], acc, 0, 0, 0);
}

// Two results, rows 0..15 and 16..31, as an operand summed over their rows
template <typename S, int PARTS> __device__ inline Frag<S, PARTS> frag_of(const f4& lo, const f4& hi) {
    Frag<S, PARTS> f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float x = j < 4 ? lo[j] : hi[j - 4];
        if constexpr (sizeof(S) == 4) {
            f.v[j] = x;
        } else {
            const bf16 h = bf16(x);
            f.p[0][j] = h;
            if constexpr (PARTS == 2) f.p[1][j] = bf16(x - float(h));
        }
    }
    return f;
}
template <int PARTS> __device__ inline const Frag<float, 1>& narrow(const Frag<float, PARTS>& f) { return f; }
template <int PARTS> __device__ inline Frag<bf16, 1> narrow(const Frag<bf16, PARTS>& f) { return {{f.p[0]}}; }

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

// Eight elements of E as they are held
template <typename E> struct Eight {
    pack<E, 8> v;
    __device__ void load(const E* at, int left) {          // left: elements up to the row's end
        if (left >= 8) v = pack<E, 8>::load(at);
        else v = pack<E, 8>::load_part(at, left < 0 ? 0 : left);
    }
    __device__ float square() const {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) s = fmaf(float(v.v[j]), float(v.v[j]), s);
        return s;
    }
    template <typename T> __device__ void put(const T& tile, int row, int c) const {
        typename Rep<E>::S x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = typename Rep<E>::S(v.v[j]);
        tile.put(row, c, x);
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
//   x     g r_k: g what a step keeps of the state before the chunk (0 past a reset), r_k one over the key's length
//   b     sigmoid(write)
//   l     l r_k: l what is left of a step's addition at the chunk's end
//   q     g r_q
//   end   what the chunk keeps of the state;  cut: a bit for each step that drops the state before it
struct Steps {
    float x[C], b[C], l[C], q[C], rk[C], rq[C], hi[C], lo[C];      // hi + lo: the logarithm of what is kept, summed up from the chunk's first step
    float end;
    uint32_t cut[2], unused;
};
template <typename S> struct Chunk {
    static constexpr int WIDE = sizeof(S) == 2 ? 2 : 1;
    S inv[WIDE][C][C], pair[WIDE][C][C];   // (I + A)^-1 and M q k^T, columns at their places
    Steps steps;
};

// Steps that a record's cut lets through: whether step j's addition is still there at step i >= j
__device__ inline int since(uint64_t cut, int i) {         // the last step up to i that drops the state, or -1
    const uint64_t m = cut & (~0ull >> (63 - i));
    return m ? 63 - __builtin_clzll(m) : -1;
}

// What the forward pass keeps for the backward pass, and what the walk backwards leaves for the gradients: two arrays of the same
// shapes, for a chunk of a value head. By columns of the state or of values, vp of them:
//   states   [vp][DK]: S before the chunk, or the gradient of S after it; rows at their places
//   steps    [vp][64]: U, or the gradient of b D; steps at their places
template <typename S> struct Kept {
    S *states, *steps;
    Kept(void* p, const Shape& s, int dk) : states(static_cast<S*>(p)), steps(states + s.B * s.G * s.chunks * int64_t(s.vp) * dk) {}
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
