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
// falls below float16's numbers is 2^-37 of that. A product's scale is a number of the lane, as a lane has one column. What is computed
// is `wide`: two float16, a value and what its rounding left, 22 bits. (Two bfloat16, without any scale, left states off by 4e-6
// and outputs in bfloat16 by 1.7 times their own rounding; the first part alone, 11 bits, left outputs and gradients in bfloat16 0.0011 off from
// the exact ones rounded, by flips to a neighbour, where both leave 0.00001 to 0.00005.) Of tensors in
// float32 the operands are float32, eight products of 16 x 16 x 4 in the place of one of 32, and scales are 1.
#pragma once
#include "pv_ops.h"

#include <type_traits>

namespace pvd {

using namespace pvo;

constexpr int C = 64;                      // steps of a chunk
constexpr int MAX_K = 128, MAX_STEP = 1 << 22;

using f4 = __attribute__((ext_vector_type(4))) float;
using h8 = __attribute__((ext_vector_type(8))) _Float16;

// What operands are held as for tensors of E; how many of those a wide one takes; lengths of keys and queries, and the scale of the
// matrices of 64 x 64, whose elements are 1 at most
template <typename E> using Rep = std::conditional_t<sizeof(E) == 2, f16, float>;
inline bool in_16_bits(int32_t dtype) { return dtype != PV_F32; }
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

// A sum over the 16 lanes of a row of columns, and over a wave; the largest over a wave
template <int N> __device__ inline int turned(int x) { return __builtin_amdgcn_mov_dpp(x, 0x120 + N, 0xf, 0xf, true); }     // by N lanes of the 16
__device__ inline float over_row(float x) {
    x += __int_as_float(turned<8>(__float_as_int(x)));
    x += __int_as_float(turned<4>(__float_as_int(x)));
    x += __int_as_float(turned<2>(__float_as_int(x)));
    return x + __int_as_float(turned<1>(__float_as_int(x)));
}
__device__ inline float sum_over_rows(float x) {           // of the four lanes that have a column
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ inline int largest_of_wave(int x) {
    x = max(x, turned<8>(x));
    x = max(x, turned<4>(x));
    x = max(x, turned<2>(x));
    x = max(x, turned<1>(x));
    auto a = __builtin_amdgcn_permlane32_swap(uint32_t(x), uint32_t(x), false, false);
    x = max(int(a[0]), int(a[1]));
    a = __builtin_amdgcn_permlane16_swap(uint32_t(x), uint32_t(x), false, false);
    return max(int(a[0]), int(a[1]));
}
// exp of a number that is not positive. Operands in 16 bits: off by |x| 2^-24 of itself, where what is left of it matters less.
template <typename S> __device__ inline float decay(float x) {
    if constexpr (sizeof(S) == 2) return __expf(x);
    return expf(x);
}
// The thread's number, of which the compiler does not know that it is the same as before: what is made from it is made where it is used,
// and no address is kept (and spilled) through a phase that has no use for it
__device__ inline int thread() {
    int id = threadIdx.x;
    asm volatile("" : "+v"(id));
    __builtin_assume(id >= 0 && id < 1024);
    return id;
}

// Nothing is moved across: the loads before it are in flight while what comes after it runs. (Left to itself the compiler puts each
// load of an operand right before its product, and a wave that is alone on its SIMD waits for every one.)
__device__ inline void fence() { __builtin_amdgcn_sched_barrier(0); }

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

// The same of products FIRST .. N - 1 with one right operand, side by side: none waits for the one before it
template <int FIRST = 0, int N, int A, int B> __device__ inline void mma_all(f4 (&acc)[N], const Frag<f16, A> (&a)[N], const Frag<f16, B>& b) {
#pragma unroll
    for (int i = A - 1; i >= 0; i--)
#pragma unroll
        for (int j = B - 1; j >= 0; j--)
            if (i + j < (A > B ? A : B))
#pragma unroll
                for (int n = FIRST; n < N; n++) acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[n].p[i], b.p[j], acc[n], 0, 0, 0);
}
template <int FIRST = 0, int N, int A, int B> __device__ inline void mma_all(f4 (&acc)[N], const Frag<float, A> (&a)[N], const Frag<float, B>& b) {
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
        for (int n = FIRST; n < N; n++) acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[n].v[j], b.v[j], acc[n], 0, 0, 0);
}

// of the first two alone
template <int A, int B, typename S> __device__ inline void mma_first(f4 (&acc)[4], const Frag<S, A> (&a)[4], const Frag<S, B>& b) {
    f4 two[2] = {acc[0], acc[1]};
    const Frag<S, A> of_two[2] = {a[0], a[1]};
    mma_all(two, of_two, b);
    acc[0] = two[0];
    acc[1] = two[1];
}

// a x; in a chunk in which some step drops the state before it (CUT), 0 where a is 0 whatever x is: what is dropped may hold anything
template <bool CUT> __device__ inline float part_of_it(float a, float x) { return CUT && a == 0.0f ? 0.0f : a * x; }
template <bool CUT> __device__ inline f4 part_of_it(const f4& a, const f4& x) {
    return f4{part_of_it<CUT>(a[0], x[0]), part_of_it<CUT>(a[1], x[1]), part_of_it<CUT>(a[2], x[2]), part_of_it<CUT>(a[3], x[3])};
}
// f(whether such a chunk it is) with that known to the compiler
template <typename F> __device__ inline void by_cut(uint64_t cuts, F&& f) {
    if (__builtin_amdgcn_readfirstlane(int(uint32_t(cuts >> 32) | uint32_t(cuts)))) f(std::true_type{});
    else f(std::false_type{});
}

// Two results, rows 0..15 and 16..31, each times a factor, as an operand summed over their rows. (The product is a float32
// before it is split: contracted into a conversion, which the compiler makes twice in two ways, its first part was now and then not the
// one that the rest is of.)
template <typename S, int PARTS> __device__ inline Frag<S, PARTS> frag_of(const f4& lo, const f4& hi, const f4& up_lo, const f4& up_hi) {
    Frag<S, PARTS> f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float x = j < 4 ? lo[j] * up_lo[j] : hi[j - 4] * up_hi[j - 4];
        if constexpr (sizeof(S) == 2) asm("" : "+v"(x));
        if constexpr (sizeof(S) == 4) {
            f.v[j] = x;
        } else {
            const f16 h = f16(x);
            f.p[0][j] = h;
            if constexpr (PARTS == 2) f.p[1][j] = f16(x - float(h));
        }
    }
    return f;
}
template <typename S, int PARTS> __device__ inline Frag<S, PARTS> frag_of(const f4& lo, const f4& hi, float up) {
    const f4 all = {up, up, up, up};
    return frag_of<S, PARTS>(lo, hi, all, all);
}

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

// A run of memory whose loads from behind its end are 0, and whose stores there are dropped: lanes that have nothing there take part
// all the same, so that no wave branches on it (a branch around a store or a load makes the next wait one for everything in flight).
constexpr uint32_t NOWHERE = 0x80000000u;
struct Buffer {
    __amdgpu_buffer_rsrc_t r;
    __device__ Buffer(const void* base, int64_t bytes) : r(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, int(bytes), 0x00027000)) {}
    template <typename T> __device__ T load(uint32_t at, int more = 0) const {
        T v;
        if constexpr (sizeof(T) == 2) { const auto x = __builtin_amdgcn_raw_buffer_load_b16(r, at, more, 0); __builtin_memcpy(&v, &x, 2); }
        if constexpr (sizeof(T) == 4) { const auto x = __builtin_amdgcn_raw_buffer_load_b32(r, at, more, 0); __builtin_memcpy(&v, &x, 4); }
        if constexpr (sizeof(T) >= 16) {
            char* to = reinterpret_cast<char*>(&v);
#pragma unroll
            for (int k = 0; k < int(sizeof(T)); k += 16) {
                const auto x = __builtin_amdgcn_raw_buffer_load_b128(r, at + k, more, 0);
                __builtin_memcpy(to + k, &x, 16);
            }
        }
        return v;
    }
    template <typename T> __device__ void store(const T& v, uint32_t at, int more = 0) const {
        if constexpr (sizeof(T) == 2) { uint16_t x; __builtin_memcpy(&x, &v, 2); __builtin_amdgcn_raw_buffer_store_b16(x, r, at, more, 0); }
        if constexpr (sizeof(T) == 4) { uint32_t x; __builtin_memcpy(&x, &v, 4); __builtin_amdgcn_raw_buffer_store_b32(x, r, at, more, 0); }
        if constexpr (sizeof(T) >= 16) {
            const char* from = reinterpret_cast<const char*>(&v);
#pragma unroll
            for (int k = 0; k < int(sizeof(T)); k += 16) {
                __attribute__((ext_vector_type(4))) uint32_t x;
                __builtin_memcpy(&x, from + k, 16);
                __builtin_amdgcn_raw_buffer_store_b128(x, r, at + k, more, 0);
            }
        }
    }
};
// `rows` rows of `n` elements of E, `stride` apart
template <typename E> __device__ inline Buffer rows_at(const E* at, int stride, int rows, int n) {
    return Buffer(at, (int64_t(rows - 1) * stride + n) * int64_t(sizeof(E)));
}

// Rows of queries or keys on their way from memory to a tile of 64 x DK, eight elements a lane. Steps past the last come out as 0 (or,
// where strides make steps overlap, as an earlier one's; their lengths are 0 in either case). A row's last eight are read as they
// lie, where K is no multiple of 8, and put one by one.
template <typename E, typename S, int DK, int THREADS> struct Rows {
    static constexpr int PER = DK / 8, COUNT = C * PER / THREADS, STEP = THREADS / PER;
    pack<E, 8> v[COUNT];
    static __device__ int column(int K) {                  // of the lane's first element
        const int c = threadIdx.x % PER * 8;
        return c + 8 <= K ? c : K >= 8 ? K - 8 : 0;
    }
    static __device__ int row(int j) { return threadIdx.x / PER + j * STEP; }
    __device__ void load(const E* at, int stride, int rows, int K) {
        const Buffer from = rows_at(at, stride, rows, K);
        const uint32_t off = (row(0) * stride + column(K)) * int(sizeof(E));
        if (K >= 8) {
#pragma unroll
            for (int j = 0; j < COUNT; j++) v[j] = from.load<pack<E, 8>>(off, j * STEP * stride * int(sizeof(E)));
        } else {
#pragma unroll
            for (int j = 0; j < COUNT; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) v[j].v[e] = from.load<E>(e < K ? off + e * uint32_t(sizeof(E)) : NOWHERE, j * STEP * stride * int(sizeof(E)));
        }
    }
    __device__ void drop(int j, bool on) { if (on) v[j].bits = typename pack<E, 8>::raw{}; }
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
    int64_t qb, qh, kb, kh, vb, vh, ab, ag, wb, wg, ob, og;        // query, key, value, gate, write, d_out: of a sequence, a head
    int32_t qt, kt, vt, at, wt, ot;                        // and of a step
    int64_t chunks;                                        // of T
    int32_t vp;                                            // V up to a multiple of 32
    float eps;
};

// What is known of a chunk's steps before its state is:
//   x     b g r: g what a step keeps of the state before the chunk (0 past a reset), r what is left of one over the key's length, b:
//   b     sigmoid(write)
//   l     l r: l what is left of a step's addition at the chunk's end
//   q     g r of the query
//   end   what the chunk keeps of the state;  cut: a bit for each step that drops the state before it
//   odd   a bit for each step whose key, gate or write is not finite, odd_query: whose query is not
struct Steps {
    float x[C], b[C], l[C], q[C], rk[C], rq[C], hi[C], lo[C];      // hi + lo: the logarithm of what is kept, summed up from the chunk's first step
    float end;
    uint32_t cut[2], odd[2], odd_query[2], unused;
};

// What one kernel leaves another lies in memory as it will lie in LDS, padding and all, and is copied there past the registers:
//   a record for each chunk of each value head: its steps, (I + A)^-1 and M q k^T, times SQUARE;
//   an image for each chunk of each key head: keys and queries.
template <typename S> struct Record {
    static constexpr int PAD = 16 / sizeof(S);
    Steps steps;
    S inv[wide_of<S>][C][C + PAD], pair[wide_of<S>][C][C + PAD];
    static constexpr int ALL = 2080 + 2 * wide_of<S> * C * (C + PAD) * int(sizeof(S));
    static constexpr int INVERSE = 2080 + wide_of<S> * C * (C + PAD) * int(sizeof(S));          // without M q k^T
    static constexpr int STRIDE = (ALL + 1023) / 1024 * 1024;
};
static_assert(sizeof(Record<f16>) == Record<f16>::ALL && sizeof(Record<float>) == Record<float>::ALL, "copied as they are");
template <typename S, int DK> constexpr int IMAGE = (2 * Tile<S, C, DK>::SIZE * int(sizeof(S)) + 1023) / 1024 * 1024;
inline uint64_t image_bytes(int32_t dk, bool half) { return (2 * 64 * (half ? (dk + 8) * 2 : (dk + 4) * 4) + 1023) / 1024 * 1024; }
template <typename S> __device__ __host__ inline char* record_of(char* work, int64_t chunk) { return work + chunk * Record<S>::STRIDE; }

// `bytes` of memory to LDS, by W waves of which this is number `wave`, 1,024 at a time (those behind the last whole kilobyte too, up to the next). Both begin at
// 16 bytes' alignment. The lanes' data goes from the memory system to LDS by itself: bring() returns at once, and the memory is there
// for a wave's own reads after arrived<N>(), N at most the number of its loads and stores since, and for the workgroup's after a barrier.
template <int W> __device__ inline void bring(const void* from, void* to, int bytes, int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE)) {
    const uint64_t base = reinterpret_cast<uint64_t>(from);
    const int last = (bytes + 1023) / 1024 - 1;
    const __attribute__((ext_vector_type(4))) int r = {__builtin_amdgcn_readfirstlane(int(base)), __builtin_amdgcn_readfirstlane(int(base >> 32)), (last + 1) * 1024,
                                                               0x00027000};
    const uint32_t lds = __builtin_amdgcn_readfirstlane(int(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)to)));
    for (int k = 0; k <= last; k += W) {   // (a wave without a kilobyte of its own copies the last one once more)
        const int at = (k + wave < last ? k + wave : last) * 1024;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds + at), "v"(threadIdx.x % WAVE * 16), "s"(r), "s"(at)
                     : "memory", "m0");
    }
}
template <int N> __device__ inline void arrived() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// Steps that a record's cut lets through: whether step j's addition is still there at step i >= j
__device__ inline int since(uint64_t cut, int i) {         // the last step up to i that drops the state, or -1
    const uint64_t m = cut & (~0ull >> (63 - i));
    return m ? 63 - __builtin_clzll(m) : -1;
}

// Steps that are not finite. The sums over a chunk's steps reach past them, where factors are 0, and 0 times NaN is NaN: so a key, query,
// gate, value or gradient of out that is not finite counts as 0 in them, and as a NaN where the recurrence takes it: forwards in the
// steps from it up to the next that drops the state, backwards in those before it down to one that drops the state.
__device__ inline bool reached(uint64_t odd, uint64_t cut, int i) {
    const int from = since(cut, i);
    return odd & (~0ull >> (63 - i)) & (~0ull << (from < 0 ? 0 : from));
}
__device__ inline bool reached_back(uint64_t odd, uint64_t cut, int i) {
    const uint64_t later = i < 63 ? cut >> (i + 1) << (i + 1) : 0;
    return odd & (~0ull << i) & (later ? (later & -later) - 1 : ~0ull);
}
// A bit for each step whose element in the lane's column is not finite, which is 0 from here on. All lanes of the wave take part.
__device__ inline uint64_t taken_out(f4 (&v)[4]) {
    uint64_t odd = 0;
#pragma unroll
    for (int it = 0; it < 4; it++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const bool on = !(fabsf(v[it][r]) < INFINITY);
            odd |= uint64_t(on) << (16 * it + r);
            v[it][r] = on ? 0.0f : v[it][r];
        }
    odd <<= thread() % WAVE / 16 * 4;
    odd |= __shfl_xor(odd, 16, WAVE);
    return odd | __shfl_xor(odd, 32, WAVE);
}
// Whether any of a lane's numbers is not finite: 0 if none
template <int N> __device__ inline float not_finite(const f4 (&v)[N]) {
    float x = 0.0f;
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) x = fmaf(0.0f, v[n][r], x);
    return x == 0.0f ? 0.0f : 1.0f;
}
// NaN over what leave() has left at `at` (nearer below): over those of the operand's places, steps first .. first + 3 and first + 16 .. first + 19, that
// f holds for. (A wave's stores to one address arrive in their order.)
template <typename S, typename B, typename F> __device__ inline void spoil(const B& to, uint32_t at, int first, F&& f) {
#pragma unroll
    for (int j = 0; j < 8; j++) to.template store<S>(S(NAN), f(first + j % 4 + j / 4 * 16) ? at + j * uint32_t(sizeof(S)) : 0x80000000u);
}

// What the forward pass keeps for the backward pass, and what the walk backwards leaves for the gradients: arrays of the same
// shapes, for a chunk of a value head, in blocks of 32 columns of the state or of values. A block is, as it will lie in LDS,
//   states   [parts][32][DK + padding]: S before the chunk, or the gradient of S after it, by columns, rows at their places
//   steps    [parts][32][64 + padding]: U, or the gradient of b D; steps at their places
// and beside the blocks scales [3][vp]: what the columns of states, of steps, and (backwards) of the gradient of out are to be multiplied by
constexpr int COLS = 32;
template <typename S, int DK> struct Kept {
    static constexpr int PAD = 16 / sizeof(S), STATE = DK + PAD, STEP = C + PAD, BLOCK = wide_of<S> * COLS * (STATE + STEP);    // elements
    static constexpr int STATES = COLS * STATE * int(sizeof(S)), STEPS = COLS * STEP * int(sizeof(S));     // of a part, in bytes
    static_assert(BLOCK * sizeof(S) % 1024 == 0, "whole kilobytes");
    S* blocks;
    float* scales;
    Kept(void* p, const Shape& s) : blocks(static_cast<S*>(p)), scales(reinterpret_cast<float*>(blocks + s.B * s.G * s.chunks * (s.vp / COLS) * int64_t(BLOCK))) {}
    // of a column's first place, in bytes; nowhere behind the last column
    static __device__ uint32_t state_at(int col, int vp) { return col < vp ? (col / COLS * BLOCK + col % COLS * STATE) * uint32_t(sizeof(S)) : NOWHERE; }
    static __device__ uint32_t step_at(int col, int vp) { return col < vp ? (col / COLS * BLOCK + col % COLS * STEP) * uint32_t(sizeof(S)) + wide_of<S> * STATES : NOWHERE; }
};
// An operand's eight places of a column to `at`, in bytes, its second part `part` behind
template <typename S, int PARTS> __device__ inline void leave(const Buffer& to, uint32_t at, const Frag<S, PARTS>& f, int part) {
    pack<S, 8> o;
#pragma unroll
    for (int k = 0; k < int(sizeof f / sizeof o); k++) {
        __builtin_memcpy(&o, reinterpret_cast<const char*>(&f) + k * sizeof o, sizeof o);
        to.store(o, at, k * part);
    }
}
inline uint64_t kept_bytes(uint64_t chunks, int32_t vp, int32_t dk, bool half) {
    const uint64_t pad = half ? 8 : 4;
    return chunks * vp * ((dk + pad + C + pad) * 4 + 12);      // (two parts of two bytes, or one of four)
}

// A lane's sixteen elements of a column of values: rows 16 it + 4 g + r. On their way each has a register of its own: two of 16 bits
// would be joined in one, which waits for both.
template <typename E> struct Sixteen {
    uint32_t v[16];
    static __device__ uint32_t first(int stride, int col, bool on) { return on ? (threadIdx.x % WAVE / 16 * 4 * stride + col) * uint32_t(sizeof(E)) : NOWHERE; }
    __device__ void load(const Buffer& from, int stride, uint32_t off) {
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int more = (16 * (j / 4) + j % 4) * stride * int(sizeof(E));
            if constexpr (sizeof(E) == 2) v[j] = __builtin_amdgcn_raw_buffer_load_b16(from.r, off, more, 0);
            else v[j] = __builtin_amdgcn_raw_buffer_load_b32(from.r, off, more, 0);
        }
    }
    static __device__ void store(const Buffer& to, int stride, uint32_t off, int j, float x) { to.store<E>(E(x), off, (16 * (j / 4) + j % 4) * stride * int(sizeof(E))); }
    static __device__ float value(uint32_t bits) {
        E e;
        __builtin_memcpy(&e, &bits, sizeof e);
        return float(e);
    }
    __device__ f4 four(int it) const { return f4{value(v[4 * it]), value(v[4 * it + 1]), value(v[4 * it + 2]), value(v[4 * it + 3])}; }
};

// The head and the columns' group of a workgroup, of `groups` to a head. Workgroups go to the eight dies in turn: those of one head
// are on one die, whose L2 then has the head's records once for all of them.
struct Part { int64_t head; int group; };
__device__ inline Part part_of(uint32_t block, int64_t heads, int groups) {
    const int64_t even = heads / 8 * 8;
    if (block >= even * groups) return {even + (block - even * groups) / groups, int((block - even * groups) % groups)};
    return {block % 8 + int64_t(8) * (block / 8 / groups), int(block / 8 % groups)};
}

// The value heads that share a query and key head are neighbours
__device__ inline int shared(const Shape& S, int g) { return g / (S.G / S.H); }

// The number of key columns that kernels are made for, K or more, and f of it
inline int32_t columns_of(int32_t K) { return K <= 32 ? 32 : K <= 64 ? 64 : 128; }
template <typename F> int32_t with_k(int32_t K, F&& f) {
    if (K <= 32) return f(std::integral_constant<int, 32>{});
    if (K <= 64) return f(std::integral_constant<int, 64>{});
    return f(std::integral_constant<int, 128>{});
}

// Sequences of few heads are walked in pieces, all at once: each from a state of zero, and beside the columns of values those of a state of
// one, which gives the map from the state before the piece to that after it; then the maps are joined from piece to piece; then each
// piece is walked once more, from its true start. There are as many pieces as give all CUs a workgroup in the first walk, of 8 chunks
// at least, as a join costs what a few chunks do; the two walks of three pieces take two thirds of the time of one over the whole.
// One sequence, heads of 128 x 128, in pieces and as one, ms: 20 heads (three pieces) of 2,048 steps 0.11 and 0.13, of 32,768 steps 1.29 and
// 1.92, in float32 3.5 and 5.8; 24 heads (two) of 2,048 steps 0.133 and 0.130, of 32,768 steps 1.84 and 2.00; 4 heads (sixteen) of 131,072
// steps 1.00 and 6.7.
struct Pieces {
    int32_t count;                         // 1: the walk is as it is
    int64_t chunks;                        // of a piece; the last one's may be fewer
};
inline Pieces pieces_of(int64_t heads, int64_t chunks, int32_t vp, int32_t dk) {
    int64_t n = 256 / (heads * ((vp + dk + 63) / 64));
    n = n < chunks / 8 ? n : chunks / 8;
    if (n < 3) return {1, chunks};
    const int64_t each = (chunks + n - 1) / n;
    return {int32_t((chunks + each - 1) / each), each};
}
// What lies in memory between them, in float32 and by columns: each piece's end from zero and, by the columns of one, its map; each
// piece's start; whether some step of the piece drops the state before it (the map is zero then, whatever that state may hold)
struct Joins {
    float *ends, *starts;
    uint32_t* cut;
    __host__ __device__ Joins(void* p, int64_t heads, int32_t pieces, int32_t vp, int32_t dk)
        : ends(static_cast<float*>(p)), starts(ends + heads * pieces * int64_t(vp + dk) * dk), cut(reinterpret_cast<uint32_t*>(starts + heads * pieces * int64_t(vp) * dk)) {}
    static uint64_t bytes(uint64_t heads, uint64_t pieces, uint64_t vp, uint64_t dk) { return heads * pieces * ((vp + dk) * dk + vp * dk + 1) * 4; }
};

constexpr int JOIN_WAVES = 4;

// ---- join_kernel: each piece's start from the one before it, in 32 bits: a workgroup for 16 columns of a head's state, of which each wave
// makes some rows of each piece, and a wave more that brings the pieces' maps to LDS, the next one while one is used. Products and
// reads of a map bound it: 2.4 us a piece of 128 x 128, 3.2 backwards. (By one wave for all rows of 16 columns 7 us, with maps read from memory by the
// waves that use them 35.)

// TURNED: backwards, each piece's end from the one after it, by the maps transposed; `ends` are of the gradient, `maps` still those of the state.
template <int DK, bool TURNED>
static __global__ __launch_bounds__((JOIN_WAVES + 1) * WAVE) void join_kernel(const float* __restrict__ state, Shape S, int pieces, Joins joins, Joins maps) {
    constexpr int KB = DK / 32, MAP = DK * DK * 4, MINE = DK / 16 > JOIN_WAVES ? DK / 16 / JOIN_WAVES : 1, ROW = DK + 4;
    __shared__ alignas(1024) char lds[2 * MAP];
    __shared__ alignas(16) float states[2][16][ROW];       // this piece's and the next one's, by columns
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), l = threadIdx.x % WAVE, grp = l / 16, m = l % 16, groups = S.vp / 16;
    const int64_t bg = blockIdx.x / groups;
    const int col = int(blockIdx.x % groups) * 16 + m, n0 = wave * MINE;
    const auto piece_of = [&](int p) { return bg * pieces + (TURNED ? pieces - 1 - p : p); };
    if (wave == JOIN_WAVES) {
        for (int p = 0; p + 1 < pieces; p++) {
            bring<1>(maps.ends + (piece_of(p) * (S.vp + DK) + S.vp) * DK, lds + p % 2 * MAP, MAP, 0);
            arrived<0>();
            __syncthreads();               // the map is there, and the one before has been used
        }
        return;
    }
    const bool on = n0 < DK / 16;          // (a whole wave)
    f4 x[MINE];
    bool cut = false;
    const auto fetch = [&](int p) {
#pragma unroll
        for (int n = 0; n < MINE; n++) if (on) x[n] = *reinterpret_cast<const f4*>(joins.ends + (piece_of(p) * (S.vp + DK) + col) * DK + 16 * (n0 + n) + 4 * grp);
        cut = maps.cut[piece_of(p)];
    };
    for (int i = threadIdx.x; i < 16 * DK; i += JOIN_WAVES * WAVE) {
        const int c = int(blockIdx.x % groups) * 16 + i % 16, d = i / 16;
        states[0][i % 16][d] = state && c < S.V && d < S.K ? state[(bg * S.K + d) * S.V + c] : 0.0f;
    }
    fetch(0);
    for (int p = 0; p + 1 < pieces; p++) {
        __syncthreads();                   // the map and the state are there, and those before them have been used
        if (!on) continue;
        const float *map = reinterpret_cast<const float*>(lds + p % 2 * MAP), *from = &states[p % 2][m][4 * grp];
        f4 z[MINE];
#pragma unroll
        for (int n = 0; n < MINE; n++) z[n] = f4{0, 0, 0, 0};
        if (!cut) {
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                Frag<float, 1> a[MINE];
#pragma unroll
                for (int n = 0; n < MINE; n++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int d = 32 * kb + 4 * grp + j % 4 + j / 4 * 16, row = 16 * (n0 + n) + m;
                        a[n].v[j] = TURNED ? map[row * DK + d] : map[d * DK + row];
                    }
                mma_all(z, a, frag_of<float, 1>(*reinterpret_cast<const f4*>(from + 32 * kb), *reinterpret_cast<const f4*>(from + 32 * kb + 16), 1.0f));
            }
        }
        float *to = joins.starts + (piece_of(p + 1) * S.vp + col) * DK + 16 * n0 + 4 * grp, *next = &states[(p + 1) % 2][m][16 * n0 + 4 * grp];
#pragma unroll
        for (int n = 0; n < MINE; n++) {
            const f4 s = z[n] + x[n];
            *reinterpret_cast<f4*>(to + 16 * n) = s;
            *reinterpret_cast<f4*>(next + 16 * n) = s;
        }
        if (p + 2 < pieces) fetch(p + 1);
    }
}

// f of the waves of a workgroup that walks over chunks forwards: four of them, 64 columns, where that makes workgroups for all CUs, else
// two. Without and with what is kept for gradients, ms, with two and with four: 64 heads of 128 x 128, 8,192 steps, bfloat16 0.66 and 0.90 against
// 0.67 and 0.94; 128 heads 1.35 and 1.76 against 0.98 and 1.67, in float32 3.46 and 3.70 against 2.54 and 3.10; 256 heads of 64 x 64, 4,096 steps, bfloat16 0.74 and
// 1.02 against 0.69 and 1.00.
template <typename F> int32_t with_waves(const Shape& S, const Pieces& pieces, F&& f) {
    if (pieces.count * S.B * S.G * ((S.vp + 63) / 64) >= 256) return f(std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, 2>{});
}

// The call's sizes and `count` strides, each of a sequence, a step and a head: of query, key, value, gate and write, or backwards of gate,
// write and d_out
inline int32_t shape_of(int64_t B, int64_t T, int32_t H, int32_t G, int32_t K, int32_t V, const int64_t* strides, int count, float eps, int32_t dtype, Shape& S, char* err,
                        size_t cap) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, cap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (B < 1 || T < 1 || H < 1 || G < H || G % H || V < 1 || V > 1 << 16)
        return fail(PV_EARG, err, cap, "shape: B, T, H >= 1, G a multiple of H, 1 <= V <= 65,536");
    if (K < 1 || K > MAX_K) return fail(PV_EARG, err, cap, "shape: 1 <= K <= 128");
    const int64_t chunks = (T + C - 1) / C, heads = B * G;
    // a launch's work items: eight waves for a chunk, or four for 32 columns of a state
    if (B >= int64_t(1) << 23 || G >= 1 << 23 || T >= int64_t(1) << 31 || heads >= int64_t(1) << 23 || heads * chunks >= int64_t(1) << 23 ||
        heads * ((V + 31) / 32) >= int64_t(1) << 23)
        return fail(PV_EARG, err, cap, "too many chunks of 64 steps, or columns of states: fewer than 2^23");
    if (!strides) return fail(PV_EARG, err, cap, "null argument");
    // (64 steps are within reach of 32-bit offsets, in bytes)
    for (int i = 1; i < count; i += 3) if (strides[i] < 0 || strides[i] > MAX_STEP) return fail(PV_EARG, err, cap, "stride: a step's is 2^22 elements at most");
    if (int64_t(G) * V > MAX_STEP || int64_t(H) * K > MAX_STEP) return fail(PV_EARG, err, cap, "shape: G V and H K are 2^22 at most");
    S = {};
    S.B = B; S.T = T; S.H = H; S.G = G; S.K = K; S.V = V; S.chunks = chunks; S.vp = (V + 31) / 32 * 32; S.eps = eps;
    const auto take = [&](int64_t& of_a_sequence, int32_t& step, int64_t& head) {
        of_a_sequence = *strides++;
        step = int32_t(*strides++);
        head = *strides++;
    };
    if (count == 15) {
        take(S.qb, S.qt, S.qh);
        take(S.kb, S.kt, S.kh);
        take(S.vb, S.vt, S.vh);
    }
    take(S.ab, S.at, S.ag);
    take(S.wb, S.wt, S.wg);
    if (count == 9) take(S.ob, S.ot, S.og);
    return PV_OK;
}

}  // namespace pvd
