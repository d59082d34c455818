// The gradients of the gated delta rule (pv_delta.hip), from those of out and of the last state.
//
// With dS the gradient of the state after a chunk, P = M Q K^T, (I + A)^-1 = T, and U, D, M, g, l as there, of a chunk
//   dU = P^T dO + l K dS,  dR = T^T dU (the gradient of b D),  dV = b dR
//   and of the state before it: g(63) dS + (g Q)^T dO - (b g K)^T dR.
// `walk_kernel` takes the chunks backwards with that, as state_kernel does forwards: it needs no state. Then every chunk by itself
// (`gradient_kernel`), with S the state before it, E = M dO U^T and F = -b M dR U^T (F below the diagonal):
//   dQ = g dO S^T + E K,  dK = l U dS^T - b g dR S^T + E^T Q + (F + F^T) K
// of keys and queries of length 1, and from there by d x = (d - x^ (x^.d)) / |x|. U of a step is b times something, so the gradient of
// write is (1 - b) dR.U of the step. The logarithm of a at step t is in M[i, j] for j < t <= i, in g(i) for i >= t, in l(j) for
// j < t, and in g(63): sums of E P' and F K' K'^T by rows and by columns, of which the pairs on one side of t cancel exactly up to
// their sums' rounding, and otherwise sums without a difference in them. The heads that share a query and key are taken one
// after another by one workgroup, so that their gradients are summed up in a fixed order.
#include "pv_delta.h"

using namespace pvd;

namespace {

constexpr int WAVES = 4, BLOCK = WAVES * WAVE;

// ---- walk_kernel: a workgroup of W waves for 16 W columns of a state's gradient

template <typename E, int DK, int W>
__global__ __launch_bounds__(W * WAVE) void walk_kernel(const E* __restrict__ query, const E* __restrict__ key, const E* __restrict__ d_out,
                                                        const float* __restrict__ d_last, Shape S, const Chunk<typename Rep<E>::S>* __restrict__ records,
                                                        E* __restrict__ d_value, float* __restrict__ d_state, Kept<typename Rep<E>::S> left_over) {
    using St = typename Rep<E>::S;
    constexpr int WIDE = Rep<E>::WIDE, ND = DK / 16, KB = DK / 32, THREADS = W * WAVE;
    using In = Tile<St, C, DK>;
    using Square = Tile<St, C, C, WIDE>;
    __shared__ alignas(16) St lds[2 * In::SIZE + 2 * Square::SIZE];
    __shared__ alignas(16) Steps st;
    const In Kt{lds}, Qt{lds + In::SIZE};
    const Square Tt{lds + 2 * In::SIZE}, Pt{lds + 2 * In::SIZE + Square::SIZE};
    const int tid = threadIdx.x, wave = tid / WAVE, l = tid % WAVE, grp = l / 16, m = l % 16;
    const int groups = (S.vp / 16 + W - 1) / W;
    const int64_t bg = blockIdx.x / groups;
    const int col = (int(blockIdx.x % groups) * W + wave) * 16 + m;
    const int64_t b = bg / S.G;
    const int g = int(bg % S.G), h = shared(S, g);
    const bool on = col < S.V;
    const E *q0 = query + b * S.qb + h * S.qh, *k0 = key + b * S.kb + h * S.kh, *o0 = d_out + b * S.ob + g * S.og + col;
    const Chunk<St>* rec = records + bg * S.chunks;

    f4 s[ND];
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 16 * n + 4 * grp + r;
            s[n][r] = d_last && on && d < S.K ? d_last[(bg * S.K + d) * S.V + col] : 0.0f;
        }

    constexpr int PER = DK / 8, IN = C * PER / THREADS, SQ = C * C * int(sizeof(St)) / 16 / THREADS, ST = (int(sizeof(Steps) / 4) + THREADS - 1) / THREADS;
    Eight<E> kp[IN], qp[IN];
    pack<St, 16 / sizeof(St)> tp[WIDE][SQ], pp[WIDE][SQ];
    float sp[ST];
    E op[16];
    auto fetch = [&](int64_t n) {
        const int64_t t0 = n * C;
        const int rows = int(S.T - t0 < C ? S.T - t0 : C);
        const E *q = q0 + t0 * S.qt, *k = k0 + t0 * S.kt, *o = o0 + t0 * S.ot;
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
            for (int w = 0; w < WIDE; w++) {
                tp[w][j] = pack<St, P>::load(inv + w * C * C + at);
                pp[w][j] = pack<St, P>::load(pair + w * C * C + at);
            }
        }
        const float* from = reinterpret_cast<const float*>(&rec[n].steps);
#pragma unroll
        for (int j = 0; j < ST; j++) if (tid + j * THREADS < int(sizeof(Steps) / 4)) sp[j] = from[tid + j * THREADS];
#pragma unroll
        for (int it = 0; it < 4; it++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = 16 * it + 4 * grp + r;
                op[4 * it + r] = on && i < rows ? o[i * S.ot] : E(0.0f);
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
            for (int w = 0; w < WIDE; w++) {
                tp[w][j].store(Tt.p + w * Square::PLANE + i * Square::ROW + c);
                pp[w][j].store(Pt.p + w * Square::PLANE + i * Square::ROW + c);
            }
        }
        float* to = reinterpret_cast<float*>(&st);
#pragma unroll
        for (int j = 0; j < ST; j++) if (tid + j * THREADS < int(sizeof(Steps) / 4)) to[tid + j * THREADS] = sp[j];
    };
    const auto four = [&](const float* p, int it) { return *reinterpret_cast<const f4*>(p + 16 * it + 4 * grp); };
    const auto leave = [&](St* to, const auto& f) {        // eight places of an operand's first part
        pack<St, 8> o;
        __builtin_memcpy(&o, &f, sizeof o);
        o.store(to);
    };

    fetch(S.chunks - 1);
    for (int64_t n = S.chunks - 1; n >= 0; n--) {
        __syncthreads();                   // the chunk after has been used
        stage();
        f4 o[4];
#pragma unroll
        for (int j = 0; j < 16; j++) o[j / 4][j % 4] = float(op[j]);
        __syncthreads();
        if (n) fetch(n - 1);
        const int64_t row = (bg * S.chunks + n) * S.vp + col;
        Frag<St, WIDE> sf[KB];
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
            sf[kb] = frag_of<St, WIDE>(s[2 * kb], s[2 * kb + 1]);
            if (col < S.vp) leave(left_over.states + row * DK + 32 * kb + 8 * grp, sf[kb]);
        }
        // dU = l K dS + P^T dO
        Frag<St, WIDE> uf[2];
        f4 u[4];
        Frag<St, 1> of[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) of[kb] = frag_of<St, 1>(o[2 * kb], o[2 * kb + 1]);      // (exact: these are tensors' elements)
#pragma unroll
        for (int it = 0; it < 4; it++) {
            f4 x = {0, 0, 0, 0};
#pragma unroll
            for (int kb = 0; kb < KB; kb++) mma(x, Kt.rows(16 * it, kb), sf[kb]);
            const f4 ls = four(st.l, it);
#pragma unroll
            for (int r = 0; r < 4; r++) u[it][r] = ls[r] == 0.0f ? 0.0f : ls[r] * x[r];
#pragma unroll
            for (int kb = it / 2; kb < 2; kb++) mma(u[it], Pt.cols(16 * it, kb), of[kb]);
            if (it % 2) uf[it / 2] = frag_of<St, WIDE>(u[it - 1], u[it]);
        }
        // dR = T^T dU
        Frag<St, WIDE> rf[2], qf[2];
        f4 d[4];
#pragma unroll
        for (int it = 0; it < 4; it++) {
            d[it] = f4{0, 0, 0, 0};
#pragma unroll
            for (int kb = it / 2; kb < 2; kb++) mma(d[it], Tt.cols(16 * it, kb), uf[kb]);
        }
        const int64_t t0 = n * C;
        E* to = d_value + ((b * S.T + t0) * S.G + g) * S.V + col;
#pragma unroll
        for (int it = 0; it < 4; it++) {
            const f4 bs = four(st.b, it);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = 16 * it + 4 * grp + r;
                if (on && t0 + i < S.T) to[int64_t(i) * S.G * S.V] = E(bs[r] * d[it][r]);
            }
        }
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            f4 x[2], y[2];
            const Frag<St, 1> df = frag_of<St, 1>(d[2 * kb], d[2 * kb + 1]);
            if (col < S.vp) leave(left_over.steps + row * C + 32 * kb + 8 * grp, df);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                x[j] = four(st.q, 2 * kb + j) * o[2 * kb + j];
                y[j] = -(four(st.b, 2 * kb + j) * four(st.x, 2 * kb + j)) * d[2 * kb + j];
            }
            qf[kb] = frag_of<St, WIDE>(x[0], x[1]);
            rf[kb] = frag_of<St, WIDE>(y[0], y[1]);
        }
        const float end = st.end;
#pragma unroll
        for (int k = 0; k < ND; k++) {
#pragma unroll
            for (int r = 0; r < 4; r++) s[k][r] = end == 0.0f ? 0.0f : end * s[k][r];
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                mma(s[k], Qt.cols(16 * k, kb), qf[kb]);
                mma(s[k], Kt.cols(16 * k, kb), rf[kb]);
            }
        }
    }
    if (!d_state) return;
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 16 * n + 4 * grp + r;
            if (on && d < S.K) d_state[(bg * S.K + d) * S.V + col] = s[n][r];
        }
}

// ---- gradient_kernel: a workgroup of four waves for each chunk of each query and key head. A wave has 16 steps' rows of every product;
// columns of values are summed over in blocks of 32, staged while the block before is used.

constexpr int BLOCK_V = 32;

__device__ inline float row16(float x) {   // a sum over the 16 lanes that have a row's columns
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) x += __shfl_xor(x, d, WAVE);
    return x;
}

template <typename E, int DK>
__global__ __launch_bounds__(BLOCK) void gradient_kernel(const E* __restrict__ query, const E* __restrict__ key, const E* __restrict__ gate, const E* __restrict__ write,
                                                         const E* __restrict__ d_out, Shape S, const Chunk<typename Rep<E>::S>* __restrict__ records,
                                                         const Kept<typename Rep<E>::S> kept, const Kept<typename Rep<E>::S> walked, E* __restrict__ d_query,
                                                         E* __restrict__ d_key, E* __restrict__ d_gate, E* __restrict__ d_write) {
    using St = typename Rep<E>::S;
    constexpr int ND = DK / 16, KB = DK / 32, PER = DK / 8;
    using In = Tile<St, C, DK>;
    using Ot = Tile<St, C, BLOCK_V>;
    using Sv = Tile<St, BLOCK_V, DK>;
    using Uv = Tile<St, BLOCK_V, C>;
    using Square = Tile<St, C, C>;
    constexpr int STAGED = Ot::SIZE + 2 * Sv::SIZE + 2 * Uv::SIZE, MORE = STAGED > 3 * Square::SIZE ? STAGED : 3 * Square::SIZE;
    __shared__ alignas(16) St lds[2 * In::SIZE + MORE];
    __shared__ alignas(16) Steps st;
    __shared__ float rows[C], columns[WAVES][C], left[C], whole[WAVES], writes[C];
    const In Kt{lds}, Qt{lds + In::SIZE};
    St* const more = lds + 2 * In::SIZE;
    const Ot Od{more};
    const Sv S0{more + Ot::SIZE}, S1{more + Ot::SIZE + Sv::SIZE};
    const Uv Us{more + Ot::SIZE + 2 * Sv::SIZE}, Rs{more + Ot::SIZE + 2 * Sv::SIZE + Uv::SIZE};
    const Square Ek{more}, Eq{more + Square::SIZE}, Ff{more + 2 * Square::SIZE};       // (once the blocks of values have been used)
    const int tid = threadIdx.x, wave = tid / WAVE, l = tid % WAVE, grp = l / 16, m = l % 16, band = 16 * wave;
    const int64_t chunk = blockIdx.x % S.chunks, bh = blockIdx.x / S.chunks;
    const int64_t b = bh / S.H, t0 = chunk * C;
    const int h = int(bh % S.H), share = S.G / S.H, steps = int(S.T - t0 < C ? S.T - t0 : C);
    const E *q0 = query + b * S.qb + t0 * S.qt + h * S.qh, *k0 = key + b * S.kb + t0 * S.kt + h * S.kh;
    for (int p = tid; p < C * PER; p += BLOCK) {
        const int i = p / PER, c = p % PER * 8, n = i < steps ? S.K - c : 0;
        Eight<E> q, k;
        q.load(q0 + i * S.qt + c, n);
        k.load(k0 + i * S.kt + c, n);
        q.put(Qt, i, c);
        k.put(Kt, i, c);
    }
    const f4 zero = {0, 0, 0, 0};
    f4 tq[ND], tk[ND];                     // the gradients of the query and the key, over the value heads so far
#pragma unroll
    for (int n = 0; n < ND; n++) tq[n] = tk[n] = zero;

    for (int j = 0; j < share; j++) {
        const int g = h * share + j;
        const int64_t at = (b * S.G + g) * S.chunks + chunk;
        const E* o0 = d_out + b * S.ob + t0 * S.ot + g * S.og;
        const St *s0 = kept.states + at * S.vp * DK, *s1 = walked.states + at * S.vp * DK, *u0 = kept.steps + at * S.vp * C, *r0 = walked.steps + at * S.vp * C;
        f4 aq[ND], from[ND], to[ND], dp[WAVES], da[WAVES];
#pragma unroll
        for (int n = 0; n < ND; n++) aq[n] = from[n] = to[n] = zero;
#pragma unroll
        for (int n = 0; n < WAVES; n++) dp[n] = da[n] = zero;
        float both = 0.0f;                 // of state and gradient, summed over all elements
        constexpr int SP = BLOCK_V * PER / BLOCK ? BLOCK_V * PER / BLOCK : 1;
        Eight<E> op;
        pack<St, 8> s0p[SP], s1p[SP], up, rp;
        auto fetch = [&](int v0) {
            op.load(o0 + (tid / 4) * S.ot + v0 + tid % 4 * 8, tid / 4 < steps ? S.V - v0 - tid % 4 * 8 : 0);
            const int v = v0 + tid / 8;
            const auto some = [](const St* p, bool on) { return on ? pack<St, 8>::load(p) : pack<St, 8>::load_part(p, 0); };
            up = some(u0 + int64_t(v) * C + tid % 8 * 8, v < S.vp);
            rp = some(r0 + int64_t(v) * C + tid % 8 * 8, v < S.vp);
#pragma unroll
            for (int k = 0; k < SP; k++) {
                const int p = tid + k * BLOCK, c = v0 + p / PER;
                const bool on = p < BLOCK_V * PER && c < S.vp;
                s0p[k] = some(s0 + int64_t(c) * DK + p % PER * 8, on);
                s1p[k] = some(s1 + int64_t(c) * DK + p % PER * 8, on);
            }
        };
        fetch(0);
        for (int v0 = 0; v0 < S.vp; v0 += BLOCK_V) {
            __syncthreads();               // what lies there has been used
            op.put(Od, tid / 4, tid % 4 * 8);
            Us.put_places(tid / 8, tid % 8 * 8, up);
            Rs.put_places(tid / 8, tid % 8 * 8, rp);
#pragma unroll
            for (int k = 0; k < SP; k++) {
                const int p = tid + k * BLOCK;
                if (p < BLOCK_V * PER) {
                    S0.put_places(p / PER, p % PER * 8, s0p[k]);
                    S1.put_places(p / PER, p % PER * 8, s1p[k]);
#pragma unroll
                    for (int c = 0; c < 8; c++) both = fmaf(float(s0p[k].v[c]), float(s1p[k].v[c]), both);
                }
            }
            if (v0 == 0) {                 // the steps' record with the first block
                const float* p = reinterpret_cast<const float*>(&records[at].steps);
                for (int k = tid; k < int(sizeof(Steps) / 4); k += BLOCK) reinterpret_cast<float*>(&st)[k] = p[k];
            }
            __syncthreads();
            if (v0 + BLOCK_V < S.vp) fetch(v0 + BLOCK_V);
            const auto of = Od.rows(band, 0);
            const auto rf = Rs.cols(band, 0), uf = Us.cols(band, 0);
#pragma unroll
            for (int n = 0; n < ND; n++) {
                const auto sf = S0.cols(16 * n, 0);
                mma(aq[n], of, sf);
                mma(from[n], rf, sf);
                mma(to[n], uf, S1.cols(16 * n, 0));
            }
#pragma unroll
            for (int n = 0; n < WAVES; n++) if (n <= wave) {
                const auto un = Us.cols(16 * n, 0);
                mma(dp[n], of, un);
                mma(da[n], rf, un);
            }
        }
        const uint64_t cuts = uint64_t(st.cut[1]) << 32 | st.cut[0];
        // what a step has of the state before the chunk and leaves after it, and its row's sums
        float gi[4], li[4], bi[4], rowsum[4], rki[4], rqi[4];
        const float last_hi = st.hi[C - 1], last_lo = st.lo[C - 1];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = band + 4 * grp + r;
            gi[r] = since(cuts, i) >= 0 ? 0.0f : expf(st.hi[i]);
            li[r] = i < since(cuts, C - 1) ? 0.0f : expf((last_hi - st.hi[i]) + (last_lo - st.lo[i]));
            bi[r] = st.b[i];
            rki[r] = st.rk[i];
            rqi[r] = st.rq[i];
            float dq = 0.0f, df = 0.0f, dt = 0.0f;
#pragma unroll
            for (int n = 0; n < ND; n++) {
                const float q = float(Qt.get(i, 16 * n + m)), k = float(Kt.get(i, 16 * n + m));
                dq = fmaf(q, aq[n][r], dq);
                df = fmaf(k, from[n][r], df);
                dt = fmaf(k, to[n][r], dt);
            }
            rowsum[r] = (gi[r] == 0.0f ? 0.0f : gi[r] * (rqi[r] * dq - bi[r] * rki[r] * df));
            dt = row16(dt);
            if (m == 0) left[i] = li[r] == 0.0f ? 0.0f : li[r] * rki[r] * dt;
#pragma unroll
            for (int n = 0; n < ND; n++) {
                tq[n][r] += gi[r] == 0.0f ? 0.0f : gi[r] * aq[n][r];
                tk[n][r] += (li[r] == 0.0f ? 0.0f : li[r] * to[n][r]) - (gi[r] == 0.0f ? 0.0f : bi[r] * gi[r] * from[n][r]);
            }
        }
        f4 kk[WAVES], qk[WAVES];
#pragma unroll
        for (int n = 0; n < WAVES; n++) kk[n] = qk[n] = zero;
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
            const auto ka = Kt.rows(band, kb), qa = Qt.rows(band, kb);
#pragma unroll
            for (int n = 0; n < WAVES; n++) if (n <= wave) {
                const auto kn = Kt.rows(16 * n, kb);
                mma(kk[n], ka, kn);
                mma(qk[n], qa, kn);
            }
        }
        both = wave_sum(both);
        if (l == 0) whole[wave] = both;
        __syncthreads();                   // the last block of values has been used
        // E and F with the lengths of what they are multiplied by, F on both sides of the diagonal
#pragma unroll
        for (int n = 0; n < WAVES; n++) {
            const int c = 16 * n + m;
            const float rk = st.rk[c], hi = st.hi[c], lo = st.lo[c];
            float column = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = band + 4 * grp + r;
                const bool on = c <= i && c >= since(cuts, i);
                float e = 0.0f, f = 0.0f;
                if (on) {
                    const float M = expf((st.hi[i] - hi) + (st.lo[i] - lo));
                    e = M * dp[n][r];
                    if (c < i) {
                        f = -M * bi[r] * da[n][r];
                        const float pair = e * rqi[r] * rk * qk[n][r] + f * rki[r] * rk * kk[n][r];
                        rowsum[r] += pair;
                        column += pair;
                    } else {
                        writes[i] = da[n][r];
                    }
                }
                Ek.p[i * Square::ROW + place(c)] = St(e * rk);
                Eq.p[i * Square::ROW + place(c)] = St(e * rqi[r]);
                if (c <= i) {
                    Ff.p[i * Square::ROW + place(c)] = St(f * rk);
                    if (c < i) Ff.p[c * Square::ROW + place(i)] = St(f * rki[r]);
                }
            }
            column += __shfl_xor(column, 16, WAVE);
            column += __shfl_xor(column, 32, WAVE);
            if (grp == 0) columns[wave][c] = column;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float x = row16(rowsum[r]);
            if (m == 0) rows[band + 4 * grp + r] = x;
        }
        __syncthreads();
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            const auto ek = Ek.rows(band, kb), eq = Eq.cols(band, kb), ff = Ff.rows(band, kb);
#pragma unroll
            for (int n = 0; n < ND; n++) {
                const auto kn = Kt.cols(16 * n, kb);
                mma(tq[n], ek, kn);
                mma(tk[n], ff, kn);
                mma(tk[n], eq, Qt.cols(16 * n, kb));
            }
        }
        if (wave == 0) {                   // a lane for each step: gates
            const auto same = [&](int i) { return i < C && since(cuts, i) <= l; };     // no step up to i, from the next on, drops the state
            double after = double(rows[l]) - (double(columns[0][l]) + columns[1][l] + columns[2][l] + columns[3][l]);
            double before = left[l];
#pragma unroll
            for (int d = 1; d < WAVE; d <<= 1) {
                const double x = __shfl_down(after, d, WAVE), y = __shfl_up(before, d, WAVE);
                if (same(l + d)) after += x;
                if (l >= d) before += y;
            }
            before = __shfl_up(before, 1, WAVE);
            if (l == 0) before = 0.0;
            const int64_t t = t0 + l;
            if (l < steps) {
                const float x = float(gate[b * S.ab + t * S.at + g * S.ag]), w = float(write[b * S.wb + t * S.wt + g * S.wg]);
                const bool first = since(cuts, l) < 0;
                double d = after + before;
                if (first && st.end != 0.0f) d += double(st.end) * (double(whole[0]) + whole[1] + whole[2] + whole[3]);
                const bool cut = cuts >> l & 1;
                d_gate[(b * S.T + t) * S.G + g] = E(cut ? 0.0f : float(-d / (1.0 + exp(-double(x)))));
                d_write[(b * S.T + t) * S.G + g] = E(writes[l] / (1.0f + expf(w)));
            }
        }
    }
    // of the query and the key themselves
    E *dq0 = d_query + ((b * S.T + t0) * S.H + h) * S.K, *dk0 = d_key + ((b * S.T + t0) * S.H + h) * S.K;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int i = band + 4 * grp + r;
        const float rk = st.rk[i], rq = st.rq[i];
        float q[ND], k[ND], dq = 0.0f, dk = 0.0f;
#pragma unroll
        for (int n = 0; n < ND; n++) {
            q[n] = float(Qt.get(i, 16 * n + m)) * rq;
            k[n] = float(Kt.get(i, 16 * n + m)) * rk;
            dq = fmaf(q[n], tq[n][r], dq);
            dk = fmaf(k[n], tk[n][r], dk);
        }
        dq = row16(dq);
        dk = row16(dk);
#pragma unroll
        for (int n = 0; n < ND; n++) {
            const int c = 16 * n + m;
            if (i < steps && c < S.K) {
                dq0[int64_t(i) * S.H * S.K + c] = E(rq * fmaf(-q[n], dq, tq[n][r]));
                dk0[int64_t(i) * S.H * S.K + c] = E(rk * fmaf(-k[n], dk, tk[n][r]));
            }
        }
    }
}

template <typename E, int DK>
int32_t backward(const void* query, const void* key, const void* gate, const void* write, const void* d_out, const float* d_last, const Shape& S, void* kept, void* records,
                 void* d_query, void* d_key, void* d_value, void* d_gate, void* d_write, float* d_state, void* work, hipStream_t stream, char* err, size_t errcap) {
    using St = typename Rep<E>::S;
    constexpr int W = 4;
    const auto in = [](const void* p) { return static_cast<const E*>(p); };
    const auto out = [](void* p) { return static_cast<E*>(p); };
    const auto* rec = static_cast<const Chunk<St>*>(records);
    const Kept<St> before(kept, S, DK), walked(work, S, DK);
    walk_kernel<E, DK, W><<<dim3(S.B * S.G * ((S.vp / 16 + W - 1) / W)), W * WAVE, 0, stream>>>(in(query), in(key), in(d_out), d_last, S, rec, out(d_value), d_state, walked);
    gradient_kernel<E, DK><<<dim3(S.B * S.H * S.chunks), BLOCK, 0, stream>>>(in(query), in(key), in(gate), in(write), in(d_out), S, rec, before, walked, out(d_query),
                                                                            out(d_key), out(d_gate), out(d_write));
    return launched(err, errcap);
}

}  // namespace

extern "C" int32_t pv_gated_delta_backward_hip(const void* query, const void* key, const void* gate, const void* write, const void* d_out, const float* d_last, int64_t B,
                                               int64_t T, int32_t H, int32_t G, int32_t K, int32_t V, const int64_t* strides, float eps, int32_t dtype, const void* kept,
                                               const void* records, void* d_query, void* d_key, void* d_value, void* d_gate, void* d_write, float* d_state, void* work,
                                               uint64_t work_bytes, void* stream, char* err, size_t errcap) {
    Shape S;
    if (int32_t e = shape_of(B, T, H, G, K, V, strides, eps, dtype, S, err, errcap)) return e;
    S.ob = strides[15];
    S.ot = strides[16];
    S.og = strides[17];
    if (S.ot < -(1 << 24) || S.ot > 1 << 24) return fail(PV_EARG, err, errcap, "stride: a step's is 2^24 elements at most");
    if (!query || !key || !gate || !write || !d_out || !kept || !records || !d_query || !d_key || !d_value || !d_gate || !d_write)
        return fail(PV_EARG, err, errcap, "null argument");
    if (!aligned(kept, 16) || !aligned(records, 16)) return fail(PV_EARG, err, errcap, "kept, records: not 16-byte aligned");
    const uint64_t need = pv_gated_delta_kept_bytes(B, T, G, K, V, dtype);
    if (!work || work_bytes < need || !aligned(work, 16)) return fail(PV_EARG, err, errcap, "work: too small, or not 16-byte aligned");
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        return with_k(K, [&](auto k) {
            return backward<E, decltype(k)::value>(query, key, gate, write, d_out, d_last, S, const_cast<void*>(kept), const_cast<void*>(records), d_query, d_key, d_value,
                                                   d_gate, d_write, d_state, work, hipStream_t(stream), err, errcap);
        });
    });
}
