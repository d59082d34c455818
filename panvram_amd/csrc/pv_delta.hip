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
template <typename S, int WIDE> __device__ inline void record(const float* m, int row, S (*to)[C][C]) {
    for (int k = threadIdx.x; k < C * C / 8; k += BLOCK) {
        const int i = k / 8, at = k % 8 * 8;                       // eight places: columns c .. c + 3 and c + 16 .. c + 19
        const int c = (at & ~31) | (at & 24) >> 1;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = m[i * row + c + j % 4 + j / 4 * 16];
        pack<S, 8> o;
#pragma unroll
        for (int w = 0; w < WIDE; w++) {
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
__global__ __launch_bounds__(BLOCK) void chunk_kernel(const E* __restrict__ query, const E* __restrict__ key, const E* __restrict__ gate, const E* __restrict__ write,
                                                      const uint8_t* __restrict__ reset, Shape S, Chunk<typename Rep<E>::S>* __restrict__ records) {
    using St = typename Rep<E>::S;
    using In = Tile<St, C, DK>;
    constexpr int ROW = C + 4, MATRIX = C * ROW * 4;
    constexpr int BYTES = 2 * In::SIZE * int(sizeof(St)) > 3 * MATRIX ? 2 * In::SIZE * int(sizeof(St)) : 3 * MATRIX;
    __shared__ alignas(16) char lds[BYTES];
    __shared__ Steps st;
    const In Kt{reinterpret_cast<St*>(lds)}, Qt{reinterpret_cast<St*>(lds) + In::SIZE};
    float *A = reinterpret_cast<float*>(lds), *P = A + C * ROW, *T = P + C * ROW;       // (once K and Q have been used)
    const int tid = threadIdx.x, wave = tid / WAVE, l = tid % WAVE, grp = l / 16, m = l % 16;
    const int64_t chunk = blockIdx.x % S.chunks, bg = blockIdx.x / S.chunks;
    const int64_t b = bg / S.G, t0 = chunk * C;
    const int g = int(bg % S.G), h = shared(S, g), rows = int(S.T - t0 < C ? S.T - t0 : C);
    // queries and keys, and one over their lengths
    constexpr int PER = DK / 8;            // packs of a row, one a lane
    const E *q0 = query + b * S.qb + t0 * S.qt + h * S.qh, *k0 = key + b * S.kb + t0 * S.kt + h * S.kh;
#pragma unroll
    for (int p = tid; p < C * PER; p += BLOCK) {
        const int i = p / PER, c = p % PER * 8;
        Eight<E> q, k;
        const int left = i < rows ? S.K - c : 0;
        q.load(q0 + i * S.qt + c, left);
        k.load(k0 + i * S.kt + c, left);
        q.put(Qt, i, c);
        k.put(Kt, i, c);
        float sq = q.square(), sk = k.square();
#pragma unroll
        for (int d = PER / 2; d; d >>= 1) { sq += __shfl_xor(sq, d, WAVE); sk += __shfl_xor(sk, d, WAVE); }
        if (p % PER == 0) {
            st.rq[i] = i < rows ? 1.0f / sqrtf(sq + S.eps) : 0.0f;
            st.rk[i] = i < rows ? 1.0f / sqrtf(sk + S.eps) : 0.0f;
        }
    }
    if (wave == 0) {                       // a lane for each step: gates, and their logarithms summed up
        const int64_t t = t0 + l;
        float la = 0.0f, beta = 0.0f;
        bool cut = false;
        if (l < rows) {
            const float x = float(gate[b * S.ab + t * S.at + g * S.ag]), w = float(write[b * S.wb + t * S.wt + g * S.wg]);
            la = -(fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))));
            if (x != x) la = x;
            beta = 1.0f / (1.0f + expf(-w));
            cut = la < -104.0f || (reset && reset[b * S.T + t]);    // (exp(-104) is 0 in 32 bits)
        }
        const uint64_t cuts = __ballot(cut);
        double c = cut ? 0.0 : double(la);
#pragma unroll
        for (int d = 1; d < WAVE; d <<= 1) {
            const double o = __shfl_up(c, d, WAVE);
            if (l >= d) c += o;
        }
        const double last = __shfl(c, C - 1, WAVE);
        const float hi = float(c);
        st.b[l] = beta;
        st.hi[l] = hi;
        st.lo[l] = float(c - double(hi));
        st.x[l] = cuts & (~0ull >> (63 - l)) ? 0.0f : expf(hi);     // (times the lengths below)
        st.l[l] = l < since(cuts, C - 1) ? 0.0f : expf(float(last - c));
        if (l == C - 1) st.end = cuts ? 0.0f : expf(hi);
        if (l < 2) st.cut[l] = uint32_t(cuts >> (32 * l));
        if (l == 0) st.unused = 0;
    }
    __syncthreads();
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
    __syncthreads();
    if (tid < C) {
        st.x[tid] = shift * st.rk[tid];
        st.q[tid] = shift * st.rq[tid];
        st.l[tid] *= st.rk[tid];
    }
#pragma unroll
    for (int j = 0; j < WAVES; j++) {
        const int col = 16 * j + m;
        const float rk = st.rk[col], hi = st.hi[col], lo = st.lo[col];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = 16 * wave + 4 * grp + r;
            const bool on = col <= i && col >= since(cuts, i);
            const float M = on ? expf((st.hi[i] - hi) + (st.lo[i] - lo)) * rk : 0.0f;
            P[i * ROW + col] = on ? M * st.rq[i] * qk[j][r] : 0.0f;
            A[i * ROW + col] = on && col < i ? M * st.rk[i] * st.b[i] * kk[j][r] : 0.0f;
            T[i * ROW + col] = 0.0f;
        }
    }
    __syncthreads();
    auto& out = records[blockIdx.x];
    constexpr int WIDE = Rep<E>::WIDE;
    if (wave == 0) {                       // the inverses of the diagonal's blocks: a lane for a column of one
        float t[16];
        const float* a = A + 16 * grp * ROW + 16 * grp;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float v = i == m ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; j++) v = fmaf(-a[i * ROW + j], t[j], v);
            t[i] = v;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) T[(16 * grp + i) * ROW + 16 * grp + m] = t[i];
    }
    record<St, WIDE>(P, ROW, out.pair);
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
    }
    __syncthreads();
    record<St, WIDE>(T, ROW, out.inv);
    const float* from = reinterpret_cast<const float*>(&st);
    float* to = reinterpret_cast<float*>(&out.steps);
    for (int k = tid; k < int(sizeof(Steps) / 4); k += BLOCK) to[k] = from[k];
}

// ---- state_kernel: a workgroup of W waves for 16 W columns of a state

template <typename E, int DK, int W>
__global__ __launch_bounds__(W * WAVE) void state_kernel(const E* __restrict__ query, const E* __restrict__ key, const E* __restrict__ value,
                                                         const float* __restrict__ state, Shape S, const Chunk<typename Rep<E>::S>* __restrict__ records,
                                                         E* __restrict__ out, float* __restrict__ last, bool keep, Kept<typename Rep<E>::S> kept) {
    using St = typename Rep<E>::S;
    constexpr int WIDE = Rep<E>::WIDE, ND = DK / 16, KB = DK / 32, THREADS = W * WAVE;
    using In = Tile<St, C, DK>;
    using Square = Tile<St, C, C, WIDE>;
    using Part = Tile<St, C, C>;
    __shared__ alignas(16) St lds[2 * In::SIZE + Square::SIZE + Part::SIZE];
    __shared__ alignas(16) Steps st;
    const In Kt{lds}, Qt{lds + In::SIZE};
    const Square Tt{lds + 2 * In::SIZE};
    const Part Pt{lds + 2 * In::SIZE + Square::SIZE};
    const int tid = threadIdx.x, wave = tid / WAVE, l = tid % WAVE, grp = l / 16, m = l % 16;
    const int groups = (S.vp / 16 + W - 1) / W;
    const int64_t bg = blockIdx.x / groups;
    const int col = (int(blockIdx.x % groups) * W + wave) * 16 + m;
    const int64_t b = bg / S.G;
    const int g = int(bg % S.G), h = shared(S, g);
    const bool on = col < S.V;
    const E *q0 = query + b * S.qb + h * S.qh, *k0 = key + b * S.kb + h * S.kh, *v0 = value + b * S.vb + g * S.vh + col;
    const Chunk<St>* rec = records + bg * S.chunks;

    f4 s[ND];
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 16 * n + 4 * grp + r;
            s[n][r] = state && on && d < S.K ? state[(bg * S.K + d) * S.V + col] : 0.0f;
        }

    // a chunk on its way from memory to LDS
    constexpr int PER = DK / 8, IN = C * PER / THREADS, SQ = C * C * int(sizeof(St)) / 16 / THREADS, ST = (int(sizeof(Steps) / 4) + THREADS - 1) / THREADS;
    Eight<E> kp[IN], qp[IN];
    pack<St, 16 / sizeof(St)> tp[WIDE][SQ], pp[SQ];
    float sp[ST];
    E vp[16];
    auto fetch = [&](int64_t n) {
        const int64_t t0 = n * C;
        const int rows = int(S.T - t0 < C ? S.T - t0 : C);
        const E *q = q0 + t0 * S.qt, *k = k0 + t0 * S.kt, *v = v0 + t0 * S.vt;
#pragma unroll
        for (int j = 0; j < IN; j++) {
            const int p = tid + j * THREADS, i = p / PER, c = p % PER * 8, left = i < rows ? S.K - c : 0;
            kp[j].load(k + i * S.kt + c, left);
            qp[j].load(q + i * S.qt + c, left);
        }
        constexpr int P = 16 / sizeof(St);
        const St *inv = &rec[n].inv[0][0][0], *pair = &rec[n].pair[0][0][0];
#pragma unroll
        for (int j = 0; j < SQ; j++) {
            const int at = (tid + j * THREADS) * P;
#pragma unroll
            for (int w = 0; w < WIDE; w++) tp[w][j] = pack<St, P>::load(inv + w * C * C + at);
            pp[j] = pack<St, P>::load(pair + at);
        }
        const float* from = reinterpret_cast<const float*>(&rec[n].steps);
#pragma unroll
        for (int j = 0; j < ST; j++) if (tid + j * THREADS < int(sizeof(Steps) / 4)) sp[j] = from[tid + j * THREADS];
#pragma unroll
        for (int it = 0; it < 4; it++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = 16 * it + 4 * grp + r;
                vp[4 * it + r] = on && i < rows ? v[i * S.vt] : E(0.0f);
            }
    };
    auto stage = [&] {
#pragma unroll
        for (int j = 0; j < IN; j++) {
            const int p = tid + j * THREADS, i = p / PER, c = p % PER * 8;
            kp[j].put(Kt, i, c);
            qp[j].put(Qt, i, c);
        }
        constexpr int P = 16 / sizeof(St);
#pragma unroll
        for (int j = 0; j < SQ; j++) {
            const int at = (tid + j * THREADS) * P, i = at / C, c = at % C;
#pragma unroll
            for (int w = 0; w < WIDE; w++) tp[w][j].store(Tt.p + w * Square::PLANE + i * Square::ROW + c);
            pp[j].store(Pt.p + i * Part::ROW + c);
        }
        float* to = reinterpret_cast<float*>(&st);
#pragma unroll
        for (int j = 0; j < ST; j++) if (tid + j * THREADS < int(sizeof(Steps) / 4)) to[tid + j * THREADS] = sp[j];
    };
    const auto four = [&](const float* p, int it) { return *reinterpret_cast<const f4*>(p + 16 * it + 4 * grp); };

    fetch(0);
    for (int64_t n = 0; n < S.chunks; n++) {
        __syncthreads();                   // the chunk before has been used
        stage();
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = float(vp[j]);
        __syncthreads();
        if (n + 1 < S.chunks) fetch(n + 1);
        Frag<St, WIDE> sf[KB];
#pragma unroll
        for (int kb = 0; kb < KB; kb++) sf[kb] = frag_of<St, WIDE>(s[2 * kb], s[2 * kb + 1]);
        const auto leave = [&](St* to, const auto& f) {    // eight places of an operand's first part
            pack<St, 8> o;
            __builtin_memcpy(&o, &f, sizeof o);
            o.store(to);
        };
        const int64_t row = (bg * S.chunks + n) * S.vp + col;
        if (keep && col < S.vp) {
#pragma unroll
            for (int kb = 0; kb < KB; kb++) leave(kept.states + row * DK + 32 * kb + 8 * grp, sf[kb]);
        }
        // D = V - g K S, then b D as an operand; out's part g Q S
        f4 o[4];
        Frag<St, WIDE> rf[2];
        f4 pairs[2];
#pragma unroll
        for (int it = 0; it < 4; it++) {
            f4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
            for (int kb = 0; kb < KB; kb++) {
                mma(x, Kt.rows(16 * it, kb), sf[kb]);
                mma(y, Qt.rows(16 * it, kb), narrow(sf[kb]));
            }
            const f4 xs = four(st.x, it), bs = four(st.b, it), qs = four(st.q, it);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                pairs[it % 2][r] = bs[r] * (v[4 * it + r] - (xs[r] == 0.0f ? 0.0f : xs[r] * x[r]));      // (a dropped state may hold anything)
                o[it][r] = qs[r] == 0.0f ? 0.0f : qs[r] * y[r];
            }
            if (it % 2) rf[it / 2] = frag_of<St, WIDE>(pairs[0], pairs[1]);
        }
        // U = (I + A)^-1 b D; out's part (M Q K^T) U; what U adds to the state
        f4 u[4];
#pragma unroll
        for (int it = 0; it < 4; it++) {
            u[it] = f4{0, 0, 0, 0};
#pragma unroll
            for (int kb = 0; kb <= it / 2; kb++) mma(u[it], Tt.rows(16 * it, kb), rf[kb]);
        }
        Frag<St, WIDE> lf[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) lf[kb] = frag_of<St, WIDE>(u[2 * kb] * four(st.l, 2 * kb), u[2 * kb + 1] * four(st.l, 2 * kb + 1));
        const float end = st.end;
#pragma unroll
        for (int k = 0; k < ND; k++) {
#pragma unroll
            for (int r = 0; r < 4; r++) s[k][r] = end == 0.0f ? 0.0f : end * s[k][r];
#pragma unroll
            for (int kb = 0; kb < 2; kb++) mma(s[k], Kt.cols(16 * k, kb), lf[kb]);
        }
        Frag<St, 1> uf[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) uf[kb] = frag_of<St, 1>(u[2 * kb], u[2 * kb + 1]);
        if (keep && col < S.vp) {
#pragma unroll
            for (int kb = 0; kb < 2; kb++) leave(kept.steps + row * C + 32 * kb + 8 * grp, uf[kb]);
        }
        const int64_t t0 = n * C;
        E* to = out + ((b * S.T + t0) * S.G + g) * S.V + col;
#pragma unroll
        for (int it = 0; it < 4; it++) {
#pragma unroll
            for (int kb = 0; kb <= it / 2; kb++) mma(o[it], Pt.rows(16 * it, kb), uf[kb]);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = 16 * it + 4 * grp + r;
                if (on && t0 + i < S.T) to[int64_t(i) * S.G * S.V] = E(o[it][r]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 16 * n + 4 * grp + r;
            if (on && d < S.K) last[(bg * S.K + d) * S.V + col] = s[n][r];
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
    pack<float, 4> s[STEP_ROWS];
#pragma unroll
    for (int j = 0; j < STEP_ROWS; j++) {
        const int d = row + 32 * j;
        const float* from = state + (bg * S.K + d) * S.V + col;
        if (state && d < S.K && left >= 4) s[j] = pack<float, 4>::load(from);
        else s[j] = pack<float, 4>::load_part(from, state && d < S.K ? left : 0);
    }
    for (int64_t t = 0; t < S.T; t++) {
        float x = 0.0f;                    // lanes 0 .. K-1: the key, lanes 128 ..: the query
        const int d0 = tid % MAX_K;
        if (d0 < S.K) x = tid < MAX_K ? float(key[b * S.kb + t * S.kt + h * S.kh + d0]) : float(query[b * S.qb + t * S.qt + h * S.qh + d0]);
        kq[tid / MAX_K][d0] = x;
        const float square = wave_sum(x * x);
        if (tid % WAVE == 0) dots[wave][0] = square;
        __syncthreads();
        const float rk = 1.0f / sqrtf(dots[0][0] + dots[1][0] + S.eps), rq = 1.0f / sqrtf(dots[2][0] + dots[3][0] + S.eps);
        const float gt = float(gate[b * S.ab + t * S.at + g * S.ag]), wt = float(write[b * S.wb + t * S.wt + g * S.wg]);
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
        const int64_t at = b * S.vb + t * S.vt + g * S.vh + col;
        E* to = out + ((b * S.T + t) * S.G + g) * S.V + col;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int n = 4 * quad + c;
            const float v = c < left ? float(value[at + c]) : 0.0f;
            const float u = beta * (v - ((sums[0][0][n] + sums[1][0][n]) + (sums[2][0][n] + sums[3][0][n])));
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

constexpr int SHORT = 8;                   // steps that are walked one by one

template <typename E, int DK>
int32_t forward(const void* query, const void* key, const void* value, const void* gate, const void* write, const float* state, const uint8_t* reset, const Shape& S,
                void* out, float* last, void* kept, void* work, hipStream_t stream, char* err, size_t errcap) {
    using St = typename Rep<E>::S;
    constexpr int W = 4;
    const auto in = [](const void* p) { return static_cast<const E*>(p); };
    auto* records = static_cast<Chunk<St>*>(work);
    const int64_t heads = S.B * S.G;
    chunk_kernel<E, DK><<<dim3(heads * S.chunks), BLOCK, 0, stream>>>(in(query), in(key), in(gate), in(write), reset, S, records);
    state_kernel<E, DK, W><<<dim3(heads * ((S.vp / 16 + W - 1) / W)), W * WAVE, 0, stream>>>(in(query), in(key), in(value), state, S, records, static_cast<E*>(out), last,
                                                                                            kept != nullptr, Kept<St>(kept, S, DK));
    return launched(err, errcap);
}

}  // namespace

extern "C" {

uint64_t pv_gated_delta_work_bytes(int64_t B, int64_t T, int32_t G, int32_t dtype, int32_t keep) {
    if (B < 1 || G < 1 || T < 1 || (T <= SHORT && !keep)) return 0;
    const uint64_t chunks = uint64_t(B) * uint64_t(G) * uint64_t((T + C - 1) / C);
    return chunks * (dtype == PV_BF16 ? sizeof(Chunk<bf16>) : sizeof(Chunk<float>));
}

uint64_t pv_gated_delta_kept_bytes(int64_t B, int64_t T, int32_t G, int32_t K, int32_t V, int32_t dtype) {
    if (B < 1 || G < 1 || T < 1 || K < 1 || V < 1) return 0;
    return uint64_t(B) * uint64_t(G) * uint64_t((T + C - 1) / C) * uint64_t((V + 15) / 16 * 16) * ((K <= 32 ? 32 : K <= 64 ? 64 : 128) + C) * (dtype == PV_BF16 ? 2 : 4);
}

int32_t pv_gated_delta_hip(const void* query, const void* key, const void* value, const void* gate, const void* write, const float* state, const uint8_t* reset,
                           int64_t B, int64_t T, int32_t H, int32_t G, int32_t K, int32_t V, const int64_t* strides, float eps, int32_t dtype, void* out, float* last,
                           void* kept, void* work, uint64_t work_bytes, void* stream, char* err, size_t errcap) {
    Shape S;
    if (int32_t e = shape_of(B, T, H, G, K, V, strides, eps, dtype, S, err, errcap)) return e;
    if (!query || !key || !value || !gate || !write || !out || !last) return fail(PV_EARG, err, errcap, "null argument");
    if (kept && !aligned(kept, 16)) return fail(PV_EARG, err, errcap, "kept: not 16-byte aligned");
    const uint64_t need = pv_gated_delta_work_bytes(B, T, G, dtype, kept != nullptr);
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
