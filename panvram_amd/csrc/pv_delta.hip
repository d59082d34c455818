// The gated delta rule: a state S [K, V] for each value head, over [B, T], and its outputs.
//
//   a = 1 - sigmoid(gate), b = sigmoid(write); q, k divided by their lengths
//   u[t] = b (v[t] - a S[t-1]^T k[t]),  S[t] = a S[t-1] + k[t] u[t]^T,  out[t] = S[t]^T q[t]
//
// Chunks of 64 steps as matrix products. With c(i) the sum of log a in a chunk, M[i, j] = exp(c(i) - c(j)) for j <= i, g(i) =
// exp(c(i)), l(i) = exp(c(63) - c(i)), all zero across a reset, and S the state before the chunk:
//   D = V - g K S,  (I + A) U = b D with A[i, j] = b(i) M[i, j] k(i).k(j) for j < i
//   out = g Q S + (M Q K^T) U,  and the state after the chunk: g(63) S + (l K)^T U.
// Two kernels: `chunk_kernel` makes (I + A)^-1 and M Q K^T of all chunks at once, `state_kernel` walks the chunks. A wave of it has
// 16 columns of a state, which no other wave needs, and all of what follows from them in registers (pv_delta.h); what the waves of a
// workgroup share of a chunk lies in LDS, and the next chunk's is loaded meanwhile.
//
// The inverse is made by substitution in blocks of 16 and by products of inverted blocks from there, in 32 bits: each is bounded as
// the inverse is, where a series of powers of A is not (keys that are alike make them grow as binomials do).
//
// Calls of few steps walk them one by one instead (`step_kernel`), the state in registers: one read and one write of it.
//
// What bounds it. bfloat16, 8 sequences of 8,192 steps, 8 heads of 128 x 128: chunk_kernel 222 us (8,192 chunks, 7 us each on a CU that has four
// at once: chains of small products), state_kernel 457 (128 chunks in a row, 3.6 us each: one wave a SIMD, half of its time in vector
// operations between products), and 628 with the 104 KB a chunk that it keeps for gradients. In float32 a chunk takes it 7 us and more: eight products of a quarter of the rate, no second buffer. step_kernel
// reads and writes 512 states of 128 x 128 in 16 us, 4.2 TB/s (18 before a step's inputs were asked for ahead of the state).
#include "pv_delta.h"

#include <algorithm>

using namespace pvd;

namespace {

// ---- chunk_kernel: one workgroup of four waves for each chunk of each value head

constexpr int WAVES = 4, BLOCK = WAVES * WAVE;

__device__ inline f4 product16(const float* a, int arow, const f4& b, f4 acc) {      // acc + a b: a 16 x 16 in memory, b a result
    const int l = threadIdx.x % WAVE;
#pragma unroll
    for (int r = 0; r < 4; r++) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[(l % 16) * arow + (l / 16) * 4 + r], b[r], acc, 0, 0, 0);
    return acc;
}
__device__ inline f4 block16(const float* b, int brow) {                             // a 16 x 16 in memory as a result
    const int l = threadIdx.x % WAVE;
    f4 v;
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] = b[((l / 16) * 4 + r) * brow + l % 16];
    return v;
}
__device__ inline void leave16(float* to, int row, const f4& v, float sign) {
    const int l = threadIdx.x % WAVE;
#pragma unroll
    for (int r = 0; r < 4; r++) to[((l / 16) * 4 + r) * row + l % 16] = sign * v[r];
}

// A matrix of 64 x 64 in LDS into a record, in parts
template <typename S> __device__ inline void record(const float* m, int row, S (*to)[C][C + Record<S>::PAD], int first, int threads) {
    for (int k = threadIdx.x - first; k < C * C / 8; k += threads) {
        const int i = k / 8, at = k % 8 * 8;                       // eight places: columns c .. c + 3 and c + 16 .. c + 19
        const int c = (at & ~31) | (at & 24) >> 1;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = SQUARE<S> * m[i * row + c + j % 4 + j / 4 * 16];
        pack<S, 8> o;
#pragma unroll
        for (int w = 0; w < wide_of<S>; w++) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                o.v[j] = S(v[j]);
                v[j] -= float(o.v[j]);
            }
            o.store(&to[w][i][at]);
        }
    }
}

template <typename E, int DK>
__global__ __launch_bounds__(BLOCK, 4) void chunk_kernel(const E* __restrict__ query, const E* __restrict__ key, const E* __restrict__ gate, const E* __restrict__ write,
                                                      const uint8_t* __restrict__ reset, Shape S, char* __restrict__ records, char* __restrict__ images) {
    using St = Rep<E>;
    using In = Tile<St, C, DK>;
    using In8 = Rows<E, St, DK, BLOCK>;
    constexpr int ROW = C + 4, MATRIX = C * ROW * 4, KEYS = 2 * In::SIZE * int(sizeof(St));
    __shared__ alignas(16) char lds[KEYS > 2 * MATRIX ? KEYS : 2 * MATRIX];
    __shared__ alignas(16) Steps st;
    const In Kt{reinterpret_cast<St*>(lds)}, Qt{reinterpret_cast<St*>(lds) + In::SIZE};
    float *A = reinterpret_cast<float*>(lds), *T = A + C * ROW;      // (once K and Q have been used; T is M Q K^T first)
    const int tid = threadIdx.x, wave = tid / WAVE, l = tid % WAVE, grp = l / 16, m = l % 16;
    const int64_t chunk = blockIdx.x % S.chunks, bg = blockIdx.x / S.chunks;
    const int64_t b = bg / S.G, t0 = chunk * C;
    const int g = int(bg % S.G), h = shared(S, g), rows = int(S.T - t0 < C ? S.T - t0 : C);
    // queries and keys, and one over their lengths
    In8 q, k;
    q.load(query + b * S.qb + t0 * S.qt + h * S.qh, S.qt, rows, S.K);
    k.load(key + b * S.kb + t0 * S.kt + h * S.kh, S.kt, rows, S.K);
    bool odd = false;                      // gate or write is not a number
    if (wave == 0) {                       // a lane for each step: gates, and their logarithms summed up
        const int64_t t = t0 + (l < rows ? l : rows - 1);
        const float x = float(gate[b * S.ab + t * S.at + g * S.ag]), w = float(write[b * S.wb + t * S.wt + g * S.wg]);
        float la = -(fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
        const bool cut = l < rows && (la < -104.0f || (reset && reset[b * S.T + t]));      // (exp(-104) is 0 in 32 bits)
        const uint64_t cuts = __ballot(cut);
        odd = l < rows && ((x != x && !cut) || w != w);
        double c = l < rows && !cut && !odd ? double(la) : 0.0;
#pragma unroll
        for (int d = 1; d < WAVE; d <<= 1) {
            const double o = __shfl_up(c, d, WAVE);
            if (l >= d) c += o;
        }
        const double last = __shfl(c, C - 1, WAVE);
        const float hi = float(c);
        st.b[l] = l < rows && !odd ? 1.0f / (1.0f + expf(-w)) : 0.0f;
        st.hi[l] = hi;
        st.lo[l] = float(c - double(hi));
        st.x[l] = cuts & (~0ull >> (63 - l)) ? 0.0f : expf(hi);     // (times the lengths below)
        st.l[l] = l < since(cuts, C - 1) ? 0.0f : expf(float(last - c));
        if (l == C - 1) st.end = cuts ? 0.0f : expf(hi);
        if (l < 2) st.cut[l] = uint32_t(cuts >> (32 * l));
        if (l == 0) st.unused = 0;
    }
    In8::clear(Qt, S.K);
    In8::clear(Kt, S.K);
#pragma unroll
    for (int j = 0; j < In8::COUNT; j++) {
        const int i = In8::row(j);
        float sq = q.square(j, S.K), sk = k.square(j, S.K);
#pragma unroll
        for (int d = In8::PER / 2; d; d >>= 1) { sq += __shfl_xor(sq, d, WAVE); sk += __shfl_xor(sk, d, WAVE); }
        const float rq = i < rows ? 1.0f / sqrtf(sq + S.eps) : 0.0f, rk = i < rows ? 1.0f / sqrtf(sk + S.eps) : 0.0f;
        const bool on_q = sq < INFINITY && rq < INFINITY, on_k = sk < INFINITY && rk < INFINITY;
        q.drop(j, !on_q);
        k.drop(j, !on_k);
        q.put(Qt, j, on_q ? length_up<St>(rq) : 0.0f, S.K);
        k.put(Kt, j, on_k ? length_up<St>(rk) : 0.0f, S.K);
        if (tid % In8::PER == 0) {
            st.rq[i] = on_q || i >= rows ? rq : NAN;
            st.rk[i] = on_k || i >= rows ? rk : NAN;
        }
    }
    __syncthreads();
    if (g % (S.G / S.H) == 0) {            // the image of keys and queries, by the first of the value heads that share them
        char* to = images + ((b * S.H + h) * S.chunks + chunk) * IMAGE<St, DK>;
        for (int i = tid * 16; i < KEYS; i += BLOCK * 16) pack<char, 16>::load(lds + i).store(to + i);
    }
    // rows 16 wave .. of K K^T and Q K^T, up to the diagonal
    f4 kk[WAVES], qk[WAVES];
#pragma unroll
    for (int j = 0; j < WAVES; j++) kk[j] = qk[j] = f4{0, 0, 0, 0};
#pragma unroll
    for (int kb = 0; kb < DK / 32; kb++) {
        const auto ka = Kt.rows(16 * wave, kb), qa = Qt.rows(16 * wave, kb);
#pragma unroll
        for (int j = 0; j < WAVES; j++) if (j <= wave) {
            const auto kj = Kt.rows(16 * j, kb);
            mma(kk[j], ka, kj);
            mma(qk[j], qa, kj);
        }
    }
    const uint64_t cuts = uint64_t(st.cut[1]) << 32 | st.cut[0];
    const float shift = tid < C ? st.x[tid] : 0.0f;
    if (wave == 0) {
        const float rk = st.rk[l], rq = st.rq[l];
        const uint64_t odds = __ballot(odd || rk != rk), queries = __ballot(rq != rq);
        if (rk != rk) st.rk[l] = st.b[l] = 0.0f;
        if (rq != rq) st.rq[l] = 0.0f;
        if (l < 2) {
            st.odd[l] = uint32_t(odds >> (32 * l));
            st.odd_query[l] = uint32_t(queries >> (32 * l));
        }
    }
    __syncthreads();
    if (tid < C) {
        st.x[tid] = st.b[tid] * (shift * length_rest<St>(st.rk[tid]));
        st.q[tid] = shift * length_rest<St>(st.rq[tid]);
        st.l[tid] *= length_rest<St>(st.rk[tid]);
    }
    float hi[4], lo[4], kf[4], qf[4];
    int from[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int i = 16 * wave + 4 * grp + r;
        hi[r] = st.hi[i];
        lo[r] = st.lo[i];
        kf[r] = length_rest<St>(st.rk[i]) * st.b[i];
        qf[r] = length_rest<St>(st.rq[i]);
        from[r] = since(cuts, i);
    }
#pragma unroll
    for (int j = 0; j < WAVES; j++) {
        const int col = 16 * j + m;
        const float rk = length_rest<St>(st.rk[col]), hc = st.hi[col], lc = st.lo[col];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = 16 * wave + 4 * grp + r;
            const bool on = j <= wave && col <= i && col >= from[r];
            const float M = on ? decay<St>((hi[r] - hc) + (lo[r] - lc)) * rk : 0.0f;
            T[i * ROW + col] = on ? M * qf[r] * qk[j][r] : 0.0f;
            A[i * ROW + col] = on && col < i ? M * kf[r] * kk[j][r] : 0.0f;
        }
    }
    __syncthreads();
    auto& out = *reinterpret_cast<Record<St>*>(record_of<St>(records, blockIdx.x));
    float t[16];
    if (wave == 0) {                       // the inverses of the diagonal's blocks: a lane for a column of one
        f4 a[16][4];
        const float* from = A + 16 * grp * ROW + 16 * grp;
#pragma unroll
        for (int i = 1; i < 16; i++)
#pragma unroll
            for (int j = 0; j < (i + 3) / 4; j++) a[i][j] = *reinterpret_cast<const f4*>(from + i * ROW + 4 * j);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float v = i == m ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; j++) v = fmaf(-a[i][j / 4][j % 4], t[j], v);
            t[i] = v;
        }
    } else {
        record<St>(T, ROW, out.pair, WAVE, BLOCK - WAVE);
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int i = 0; i < 16; i++) T[(16 * grp + i) * ROW + 16 * grp + m] = t[i];
    } else {                               // nothing above the diagonal's blocks
        for (int k = tid - WAVE; k < C * C / 4; k += BLOCK - WAVE) {
            const int i = k / 16, c = k % 16 * 4;
            if (c / 16 > i / 16) *reinterpret_cast<f4*>(T + i * ROW + c) = f4{0, 0, 0, 0};
        }
    }
    __syncthreads();
    const auto at = [&](float* p, int i, int j) { return p + 16 * i * ROW + 16 * j; };
    const f4 zero = {0, 0, 0, 0};
    if (wave < 2) {                        // blocks (1, 0) and (3, 2)
        const int i = 2 * wave + 1;
        const f4 y = product16(at(A, i, i - 1), ROW, block16(at(T, i - 1, i - 1), ROW), zero);
        leave16(at(T, i, i - 1), ROW, product16(at(T, i, i), ROW, y, zero), -1.0f);
    }
    __syncthreads();
    if (wave < 2) {                        // blocks (2, wave) and (3, wave)
        f4 y2 = zero, y3 = zero;
        for (int k = wave; k < 2; k++) {
            const f4 t = block16(at(T, k, wave), ROW);
            y2 = product16(at(A, 2, k), ROW, t, y2);
            y3 = product16(at(A, 3, k), ROW, t, y3);
        }
        leave16(at(T, 2, wave), ROW, product16(at(T, 2, 2), ROW, y2, zero), -1.0f);
        leave16(at(T, 3, wave), ROW, product16(at(T, 3, 3), ROW, y3, product16(at(T, 3, 2), ROW, y2, zero)), -1.0f);
    } else {
        const float* from = reinterpret_cast<const float*>(&st);
        float* to = reinterpret_cast<float*>(&out.steps);
        for (int k = tid - 2 * WAVE; k < int(sizeof(Steps) / 4); k += BLOCK - 2 * WAVE) to[k] = from[k];
    }
    __syncthreads();
    record<St>(T, ROW, out.inv, 0, BLOCK);
}

// ---- state_kernel: a workgroup of W waves for 16 W columns of a state, and a wave more that brings chunks to LDS: while the one before is
// worked on, where two have room (tensors of 16 bits), else one after another. (A wave that brings is held up until the memory system
// has taken all it asks for, 3 us a chunk.)

// MAP: the first walk of a sequence in pieces; there are no outputs, and DK columns more that begin as those of one.
template <typename E, int DK, int W, bool KEEP, bool MAP>
__global__ __launch_bounds__((W + 1) * WAVE) __attribute__((amdgpu_waves_per_eu(1, 2))) void state_kernel(
    const E* __restrict__ value, const float* __restrict__ state, Shape S, const char* __restrict__ records, const char* __restrict__ images, E* __restrict__ out,
    float* __restrict__ last, Kept<Rep<E>, DK> kept, Pieces pieces, Joins joins) {
    using St = Rep<E>;
    using Ke = Kept<St, DK>;
    constexpr int WIDE = wide_of<St>, ND = DK / 16, KB = DK / 32;
    using In = Tile<St, C, DK>;
    using Square = Tile<St, C, C, WIDE>;
    using Re = Record<St>;
    constexpr int RECORD = MAP ? Re::INVERSE : Re::ALL;
    constexpr int BUFFERS = sizeof(St) == 2 ? 2 : 1, IN = IMAGE<St, DK>, BUFFER = IN + (RECORD + 1023) / 1024 * 1024;
    __shared__ alignas(1024) char lds[BUFFERS * BUFFER];
    const int tid = threadIdx.x, wave = tid / WAVE, l = tid % WAVE, grp = l / 16, m = l % 16;
    const int width = MAP ? S.vp + DK : S.vp, groups = (width / 16 + W - 1) / W;
    const auto [piece, group] = part_of(blockIdx.x, S.B * S.G * pieces.count, groups);
    const int col = (group * W + wave) * 16 + m;
    const int64_t bg = piece / pieces.count, b = bg / S.G, first = piece % pieces.count * pieces.chunks;
    const int64_t behind = first + pieces.chunks < S.chunks ? first + pieces.chunks : S.chunks;
    const int g = int(bg % S.G), h = shared(S, g);
    const bool on = col < S.V;
    const E* v0 = value + b * S.vb + g * S.vh;
    const char *rec0 = records + bg * S.chunks * Re::STRIDE, *in0 = images + (b * S.H + h) * S.chunks * IN;
    const int ot = S.G * S.V;              // steps of out
    const uint32_t value_at = Sixteen<E>::first(S.vt, col, on), out_at = Sixteen<E>::first(ot, col, on);
    const uint32_t state_at = Ke::state_at(col, S.vp) + 8 * grp * sizeof(St), step_at = Ke::step_at(col, S.vp) + 8 * grp * sizeof(St);

    f4 s[ND];
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 16 * n + 4 * grp + r;
            if constexpr (MAP) s[n][r] = col - S.vp == d ? 1.0f : 0.0f;
            else if (first) s[n][r] = col < S.vp ? joins.starts[(piece * S.vp + col) * DK + d] : 0.0f;
            else s[n][r] = state && on && d < S.K ? state[(bg * S.K + d) * S.V + col] : 0.0f;
        }
    const auto rows_of = [&](int64_t n) { return int(S.T - n * C < C ? S.T - n * C : C); };
    if (wave == W) {
        for (int64_t n = first; n < behind; n++) {
            if (n != first && BUFFERS == 1) __syncthreads();   // the chunk before has been used
            char* to = lds + (BUFFERS == 2 ? int(n & 1) * BUFFER : 0);
            bring<1>(in0 + n * IN, to, (MAP ? 1 : 2) * In::SIZE * int(sizeof(St)), 0);
            bring<1>(rec0 + n * Re::STRIDE, to + IN, RECORD, 0);
            arrived<0>();
            __syncthreads();               // the chunk is there (and of two, the one before has been used)
        }
        return;
    }
    Sixteen<E> vp;
    vp.load(rows_at(v0 + first * C * S.vt, S.vt, rows_of(first), S.V), S.vt, value_at);
    uint64_t any = 0;                      // step that drops the state before it
    for (int64_t n = first; n < behind; n++) {
        if (n != first && BUFFERS == 1) __syncthreads();
        __syncthreads();
        char* here = lds + (BUFFERS == 2 ? int(n & 1) * BUFFER : 0);
        const In Kt{reinterpret_cast<St*>(here)}, Qt{reinterpret_cast<St*>(here) + In::SIZE};
        const Re& re = *reinterpret_cast<const Re*>(here + IN);
        const Steps& st = re.steps;
        const Square Tt{const_cast<St*>(&re.inv[0][0][0])}, Pt{const_cast<St*>(&re.pair[0][0][0])};
        const auto four = [&](const float* p, int it) { return *reinterpret_cast<const f4*>(p + 16 * it + 4 * grp); };
        const uint64_t cuts = uint64_t(st.cut[1]) << 32 | st.cut[0];
        f4 v[4];
#pragma unroll
        for (int it = 0; it < 4; it++) v[it] = vp.four(it);
        any |= cuts;
        uint64_t odd = uint64_t(st.odd[1]) << 32 | st.odd[0];
        const bool some = __builtin_amdgcn_readfirstlane(st.odd[0] | st.odd[1] | st.odd_query[0] | st.odd_query[1]) || __any(not_finite(v) != 0.0f);
        if (some) odd |= taken_out(v) & (~0ull >> (C - rows_of(n)));       // (where steps overlap, one behind the last reads an earlier one's)
        bool lost = false;                 // the state before a chunk in which some step drops it is not finite
        by_cut(cuts, [&](auto cut) {
            if constexpr (decltype(cut)::value) {      // (zero times it would reach the steps that it is dropped at: it is zero, and the steps before are NaN)
                lost = over_column(not_finite(s)) != 0.0f;
#pragma unroll
                for (int k = 0; k < ND; k++)
#pragma unroll
                    for (int r = 0; r < 4; r++) s[k][r] = lost ? 0.0f : s[k][r];
            }
        });
        if (n + 1 < behind) vp.load(rows_at(v0 + (n + 1) * C * S.vt, S.vt, rows_of(n + 1), S.V), S.vt, value_at);
        const int64_t at = (bg * S.chunks + n) * S.vp;     // of the chunk in what is kept
        const Buffer blocks(kept.blocks + at / COLS * Ke::BLOCK, KEEP ? int64_t(S.vp / COLS) * Ke::BLOCK * int(sizeof(St)) : 0);
        // operands of a stage's products are loaded while the stage before runs
        Frag<St, 1> ka[KB][4], qa[KB][4], kc[2][ND];
        Frag<St, WIDE> ta[2][4], pa[2][4], sf[KB];
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int it = 0; it < 4; it++) ka[kb][it] = Kt.rows(16 * it, kb);
        fence();
        const Scale ss = scale_of<St>(over_column(largest(s)));
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
            sf[kb] = frag_of<St, WIDE>(s[2 * kb], s[2 * kb + 1], ss.up);
            if constexpr (KEEP) leave(blocks, state_at + 32 * kb * sizeof(St), sf[kb], Ke::STATES);
        }
        fence();
        if constexpr (!MAP) {
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
#pragma unroll
                for (int it = 0; it < 4; it++) qa[kb][it] = Qt.rows(16 * it, kb);
        }
        // D = V - g K S, then b D; g Q S for out
        f4 x[4], y[4], d[4];
#pragma unroll
        for (int it = 0; it < 4; it++) x[it] = y[it] = f4{0, 0, 0, 0};
#pragma unroll
        for (int kb = 0; kb < KB; kb++) mma_all(x, ka[kb], sf[kb]);
        fence();
#pragma unroll
        for (int it = 0; it < 4; it++)
#pragma unroll
            for (int kb = 0; kb <= it / 2; kb++) ta[kb][it] = Tt.rows(16 * it, kb);
#pragma unroll
        for (int kb = 0; kb < KB; kb++) if constexpr (!MAP) mma_all(y, qa[kb], sf[kb]);
        by_cut(cuts, [&](auto cut) {
#pragma unroll
            for (int it = 0; it < 4; it++) d[it] = four(st.b, it) * v[it] - part_of_it<decltype(cut)::value>(four(st.x, it) * ss.down, x[it]);
        });
        const Scale ds = scale_of<St>(over_column(largest(d)));
        Frag<St, WIDE> df[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) df[kb] = frag_of<St, WIDE>(d[2 * kb], d[2 * kb + 1], ds.up);
        fence();
        // U = (I + A)^-1 b D
#pragma unroll
        for (int k = 0; k < ND; k++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++) kc[kb][k] = Kt.cols(16 * k, kb);
        f4 u[4];
#pragma unroll
        for (int it = 0; it < 4; it++) u[it] = f4{0, 0, 0, 0};
        mma_all(u, ta[0], df[0]);
        mma_all<2>(u, ta[1], df[1]);
        const float du = ds.down * (1.0f / SQUARE<St>);        // of u
        // what it adds to the state (l r is 2 / LONG at most)
        const Scale us = scale_of<St>(over_column(largest(u)) * du);
        Frag<St, WIDE> uf[2], lf[2];
        const float up = sizeof(St) == 2 ? du * us.up : 1.0f;
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            uf[kb] = frag_of<St, WIDE>(u[2 * kb], u[2 * kb + 1], up);
            lf[kb] = frag_of<St, WIDE>(u[2 * kb], u[2 * kb + 1], four(st.l, 2 * kb) * (LONG<St> * up), four(st.l, 2 * kb + 1) * (LONG<St> * up));
            if constexpr (KEEP) leave(blocks, step_at + 32 * kb * sizeof(St), uf[kb], Ke::STEPS);
        }
        if constexpr (KEEP) {
            const Buffer scales(kept.scales + 3 * at, 3 * int64_t(S.vp) * 4);
            const uint32_t to = grp == 0 && col < S.vp ? col * 4 : NOWHERE;
            scales.store(ss.down, to);
            scales.store(us.down, to, S.vp * 4);
        }
        fence();
        if constexpr (!MAP) {
#pragma unroll
            for (int it = 0; it < 4; it++)
#pragma unroll
                for (int kb = 0; kb <= it / 2; kb++) pa[kb][it] = Pt.rows(16 * it, kb);
        }
        const float end = st.end, dl = us.down * (1.0f / LONG<St>), dp = us.down * (1.0f / SQUARE<St>);
        f4 z[ND], w[4];
#pragma unroll
        for (int k = 0; k < ND; k++) z[k] = f4{0, 0, 0, 0};
#pragma unroll
        for (int kb = 0; kb < 2; kb++) mma_all(z, kc[kb], lf[kb]);
        fence();
        // out = g Q S + (M Q K^T) U
#pragma unroll
        for (int it = 0; it < 4; it++) w[it] = f4{0, 0, 0, 0};
        if constexpr (!MAP) {
            mma_all(w, pa[0], uf[0]);
            mma_all<2>(w, pa[1], uf[1]);
        }
        by_cut(cuts, [&](auto cut) {
            constexpr bool CUT = decltype(cut)::value;
#pragma unroll
            for (int k = 0; k < ND; k++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[k][r] = fmaf(dl, z[k][r], part_of_it<CUT>(end, s[k][r]));
#pragma unroll
            for (int it = 0; it < 4; it++) if constexpr (!MAP) {
                y[it] = part_of_it<CUT>(four(st.q, it) * ss.down, y[it]);
#pragma unroll
                for (int r = 0; r < 4; r++) if (CUT && lost && 16 * it + 4 * grp + r < __builtin_ctzll(cuts)) y[it][r] = NAN;
            }
        });
        if (some) {
            const int first = thread() % WAVE / 16 * 4;
            if (reached(odd, cuts, C - 1))
#pragma unroll
                for (int k = 0; k < ND; k++) s[k] = f4{NAN, NAN, NAN, NAN};
            const uint64_t queries = uint64_t(st.odd_query[1]) << 32 | st.odd_query[0];
#pragma unroll
            for (int it = 0; it < 4; it++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = 16 * it + first + r;
                    if (reached(odd, cuts, i) || queries >> i & 1) y[it][r] = NAN;
                }
        }
        if constexpr (KEEP) if (some || __any(lost)) {     // (the gradients take from these what is NaN; their own products are by steps and heads)
            const int first = thread() % WAVE / 16 * 4;
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
                spoil<St>(blocks, step_at + 32 * kb * sizeof(St), 32 * kb + first, [&](int i) { return reached(odd, cuts, i) || (lost && i < __builtin_ctzll(cuts)); });
#pragma unroll
            for (int kb = 0; kb < KB; kb++)
                spoil<St>(blocks, state_at + 32 * kb * sizeof(St), 0, [&](int) { return lost; });
        }
        if constexpr (MAP) continue;
        const Buffer to = rows_at(out + ((b * S.T + n * C) * S.G + g) * S.V, ot, rows_of(n), S.V);
#pragma unroll
        for (int it = 0; it < 4; it++) {
#pragma unroll
            for (int r = 0; r < 4; r++) Sixteen<E>::store(to, ot, out_at, 4 * it + r, fmaf(dp, w[it][r], y[it][r]));
        }
    }
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 16 * n + 4 * grp + r;
            if (!MAP && on && d < S.K && behind == S.chunks) last[(bg * S.K + d) * S.V + col] = s[n][r];
        }
    if constexpr (MAP) {
        if (col < width) {
            float* to = joins.ends + (piece * width + col) * DK + 4 * grp;
#pragma unroll
            for (int n = 0; n < ND; n++) *reinterpret_cast<f4*>(to + 16 * n) = s[n];
        }
        if (group == 0 && tid == 0) joins.cut[piece] = any != 0;
    }
}

// ---- step_kernel: few steps, one by one. A workgroup has 32 columns of a state, a lane four neighbouring ones of every 32nd row

constexpr int STEP_COLS = 32, STEP_ROWS = MAX_K / 32;

template <typename E>
__global__ __launch_bounds__(BLOCK) void step_kernel(const E* __restrict__ query, const E* __restrict__ key, const E* __restrict__ value, const E* __restrict__ gate,
                                                     const E* __restrict__ write, const float* __restrict__ state, const uint8_t* __restrict__ reset, Shape S,
                                                     E* __restrict__ out, float* __restrict__ last) {
    __shared__ float kq[2][MAX_K], dots[WAVES][3], sums[WAVES][2][STEP_COLS];
    const int tid = threadIdx.x, wave = tid / WAVE, quad = tid % 8, row = tid / 8;
    const int groups = (S.V + STEP_COLS - 1) / STEP_COLS;
    const int64_t bg = blockIdx.x / groups, b = bg / S.G;
    const int g = int(bg % S.G), h = shared(S, g), col = int(blockIdx.x % groups) * STEP_COLS + 4 * quad;
    const int left = S.V - col;            // columns up to the state's last
    // what a step brings is asked for a step ahead, and the first before the state
    E x0 = E(0.0f), v0[4], gate0, write0;  // (x0 of lanes 0 .. K-1: the key, of lanes 128 ..: the query)
    const int d0 = tid % MAX_K;
    const auto fetch = [&](int64_t t) {
        if (d0 < S.K) x0 = tid < MAX_K ? key[b * S.kb + t * S.kt + h * S.kh + d0] : query[b * S.qb + t * S.qt + h * S.qh + d0];
        gate0 = gate[b * S.ab + t * S.at + g * S.ag];
        write0 = write[b * S.wb + t * S.wt + g * S.wg];
        const int64_t at = b * S.vb + t * S.vt + g * S.vh + col;
#pragma unroll
        for (int c = 0; c < 4; c++) v0[c] = c < left ? value[at + c] : E(0.0f);
    };
    fetch(0);
    pack<float, 4> s[STEP_ROWS];
#pragma unroll
    for (int j = 0; j < STEP_ROWS; j++) {
        const int d = row + 32 * j;
        const float* from = state + (bg * S.K + d) * S.V + col;
        if (state && d < S.K && left >= 4) s[j] = pack<float, 4>::load(from);
        else s[j] = pack<float, 4>::load_part(from, state && d < S.K ? left : 0);
    }
    for (int64_t t = 0; t < S.T; t++) {
        const float x = float(x0), gt = float(gate0), wt = float(write0);
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = float(v0[c]);
        if (t + 1 < S.T) fetch(t + 1);
        kq[tid / MAX_K][d0] = x;
        const float square = wave_sum(x * x);
        if (tid % WAVE == 0) dots[wave][0] = square;
        __syncthreads();
        const float rk = 1.0f / sqrtf(dots[0][0] + dots[1][0] + S.eps), rq = 1.0f / sqrtf(dots[2][0] + dots[3][0] + S.eps);
        const float a = 1.0f / (1.0f + expf(gt)), beta = 1.0f / (1.0f + expf(-wt));
        const bool cut = a == 0.0f || (reset && reset[b * S.T + t]);
        float sk[4] = {0, 0, 0, 0}, sq[4] = {0, 0, 0, 0}, kd[STEP_ROWS], together = 0.0f;
#pragma unroll
        for (int j = 0; j < STEP_ROWS; j++) {
            const int d = row + 32 * j;
            kd[j] = kq[0][d] * rk;
            const float qd = kq[1][d] * rq;
            together = fmaf(kd[j], qd, together);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                s[j].v[c] = cut ? 0.0f : a * s[j].v[c];
                sk[c] = fmaf(kd[j], s[j].v[c], sk[c]);
                sq[c] = fmaf(qd, s[j].v[c], sq[c]);
            }
        }
#pragma unroll
        for (int d = 8; d < WAVE; d <<= 1) {
            together += __shfl_xor(together, d, WAVE);
#pragma unroll
            for (int c = 0; c < 4; c++) { sk[c] += __shfl_xor(sk[c], d, WAVE); sq[c] += __shfl_xor(sq[c], d, WAVE); }
        }
        if (tid % WAVE < 8) {
            dots[wave][1] = together;
#pragma unroll
            for (int c = 0; c < 4; c++) { sums[wave][0][4 * quad + c] = sk[c]; sums[wave][1][4 * quad + c] = sq[c]; }
        }
        __syncthreads();
        const float kdq = (dots[0][1] + dots[1][1]) + (dots[2][1] + dots[3][1]);
        E* to = out + ((b * S.T + t) * S.G + g) * S.V + col;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int n = 4 * quad + c;
            const float u = beta * (v[c] - ((sums[0][0][n] + sums[1][0][n]) + (sums[2][0][n] + sums[3][0][n])));
            const float o = fmaf(kdq, u, (sums[0][1][n] + sums[1][1][n]) + (sums[2][1][n] + sums[3][1][n]));
            if (row == 0 && c < left) to[c] = E(o);
#pragma unroll
            for (int j = 0; j < STEP_ROWS; j++) s[j].v[c] = fmaf(kd[j], u, s[j].v[c]);
        }
    }
#pragma unroll
    for (int j = 0; j < STEP_ROWS; j++) {
        const int d = row + 32 * j;
        if (d >= S.K) continue;
        float* to = last + (bg * S.K + d) * S.V + col;
        if (left >= 4) s[j].store(to);
        else s[j].store_part(to, left);
    }
}
}  // namespace

// ---- the C entries

namespace {

// Calls of so few steps walk them one by one, where nothing is kept for gradients. Heads of 128 x 128, us: 4 heads 5.3 for one step and
// 18.4 for eight, in chunks 21.0 for nine and 21.3 for sixty-four; 512 heads 16.0, 53.6, 56.1 and 59.1.
constexpr int SHORT = 8;

template <typename E, int DK>
int32_t forward(const void* query, const void* key, const void* value, const void* gate, const void* write, const float* state, const uint8_t* reset, const Shape& S,
                void* out, float* last, void* kept, void* work, hipStream_t stream, char* err, size_t errcap) {
    using St = Rep<E>;
    const auto in = [](const void* p) { return static_cast<const E*>(p); };
    const int64_t heads = S.B * S.G;
    char *records = static_cast<char*>(work), *images = records + heads * S.chunks * Record<St>::STRIDE;
    chunk_kernel<E, DK><<<dim3(heads * S.chunks), BLOCK, 0, stream>>>(in(query), in(key), in(gate), in(write), reset, S, records, images);
    const Kept<St, DK> to(kept, S);
    const Pieces pieces = pieces_of(heads, S.chunks, S.vp, DK);
    const Joins joins(images + S.B * S.H * S.chunks * IMAGE<St, DK>, heads, pieces.count, S.vp, DK);
    if (pieces.count > 1) {
        constexpr int W = 4;
        state_kernel<E, DK, W, false, true><<<dim3(heads * pieces.count * (((S.vp + DK) / 16 + W - 1) / W)), (W + 1) * WAVE, 0, stream>>>(
            in(value), nullptr, S, records, images, nullptr, nullptr, to, pieces, joins);
        join_kernel<DK, false><<<dim3(heads * (S.vp / 16)), (JOIN_WAVES + 1) * WAVE, 0, stream>>>(state, S, pieces.count, joins, joins);
    }
    return with_waves(S, pieces, [&](auto w) {
        constexpr int W = decltype(w)::value;
        const dim3 grid(heads * pieces.count * ((S.vp / 16 + W - 1) / W));
        const auto walk = [&](auto keep) {
            state_kernel<E, DK, W, decltype(keep)::value, false><<<grid, (W + 1) * WAVE, 0, stream>>>(in(value), state, S, records, images, static_cast<E*>(out), last, to,
                                                                                                      pieces, joins);
        };
        if (kept) walk(std::true_type{});
        else walk(std::false_type{});
        return launched(err, errcap);
    });
}

}  // namespace

extern "C" {

uint64_t pv_gated_delta_work_bytes(int64_t B, int64_t T, int32_t H, int32_t G, int32_t K, int32_t V, int32_t dtype, int32_t keep) {
    if (B < 1 || H < 1 || G < 1 || T < 1 || K < 1 || V < 1 || (T <= SHORT && !keep)) return 0;
    const int64_t chunks = (T + C - 1) / C, heads = B * G;
    const int32_t vp = (V + 31) / 32 * 32, dk = columns_of(K);
    const Pieces pieces = pieces_of(heads, chunks, vp, dk);
    const bool half = in_16_bits(dtype);
    return uint64_t(B) * chunks * (uint64_t(G) * (half ? Record<f16>::STRIDE : Record<float>::STRIDE) + uint64_t(H) * image_bytes(dk, half)) +
           (pieces.count > 1 ? Joins::bytes(heads, pieces.count, vp, dk) : 0);
}

uint64_t pv_gated_delta_kept_bytes(int64_t B, int64_t T, int32_t G, int32_t K, int32_t V, int32_t dtype) {
    if (B < 1 || G < 1 || T < 1 || K < 1 || V < 1) return 0;
    return kept_bytes(uint64_t(B) * uint64_t(G) * uint64_t((T + C - 1) / C), (V + 31) / 32 * 32, columns_of(K), in_16_bits(dtype));
}

uint64_t pv_gated_delta_backward_work_bytes(int64_t B, int64_t T, int32_t G, int32_t K, int32_t V, int32_t dtype) {
    const uint64_t kept = pv_gated_delta_kept_bytes(B, T, G, K, V, dtype);
    if (!kept) return 0;
    const int32_t vp = (V + 31) / 32 * 32, dk = columns_of(K);
    const Pieces pieces = pieces_of(B * G, (T + C - 1) / C, vp, dk);
    return kept + (pieces.count > 1 ? Joins::bytes(B * G, pieces.count, vp, dk) : 0);
}

int32_t pv_gated_delta_hip(const void* query, const void* key, const void* value, const void* gate, const void* write, const float* state, const uint8_t* reset,
                           int64_t B, int64_t T, int32_t H, int32_t G, int32_t K, int32_t V, const int64_t* strides, float eps, int32_t dtype, void* out, float* last,
                           void* kept, void* work, uint64_t work_bytes, void* stream, char* err, size_t errcap) {
    Shape S;
    if (int32_t e = shape_of(B, T, H, G, K, V, strides, 15, eps, dtype, S, err, errcap)) return e;
    if (!query || !key || !value || !gate || !write || !out || !last) return fail(PV_EARG, err, errcap, "null argument");
    if (kept && !aligned(kept, 16)) return fail(PV_EARG, err, errcap, "kept: not 16-byte aligned");
    const uint64_t need = pv_gated_delta_work_bytes(B, T, H, G, K, V, dtype, kept != nullptr);
    if (need && (!work || work_bytes < need || !aligned(work, 16))) return fail(PV_EARG, err, errcap, "work: too small, or not 16-byte aligned");
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        const auto in = [](const void* p) { return static_cast<const E*>(p); };
        if (!need) {
            step_kernel<E><<<dim3(B * G * ((V + STEP_COLS - 1) / STEP_COLS)), BLOCK, 0, hipStream_t(stream)>>>(
                in(query), in(key), in(value), in(gate), in(write), state, reset, S, static_cast<E*>(out), last);
            return launched(err, errcap);
        }
        return with_k(K, [&](auto k) {
            return forward<E, decltype(k)::value>(query, key, value, gate, write, state, reset, S, out, last, kept, work, hipStream_t(stream), err, errcap);
        });
    });
}

}  // extern "C"
