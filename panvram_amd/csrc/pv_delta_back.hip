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
                                                        E* __restrict__ d_value, float* __restrict__ d_state, Kept<typename Rep<E>::S> walked) {
    using St = typename Rep<E>::S;
    constexpr int WIDE = wide_of<St>, ND = DK / 16, KB = DK / 32, THREADS = W * WAVE;
    using In = Tile<St, C, DK>;
    using Square = Tile<St, C, C, WIDE>;
    using In8 = Rows<E, DK, THREADS>;
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
    const bool on = col < S.V, held = col < S.vp;
    const E *q0 = query + b * S.qb + h * S.qh, *k0 = key + b * S.kb + h * S.kh, *o0 = d_out + b * S.ob + g * S.og + (on ? col : S.V - 1);
    const Chunk<St>* rec = records + bg * S.chunks;

    f4 s[ND];
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 16 * n + 4 * grp + r;
            s[n][r] = d_last && on && d < S.K ? d_last[(bg * S.K + d) * S.V + col] : 0.0f;
        }

    In8 qp, kp;
    float qr[In8::COUNT], kr[In8::COUNT];
    SquareOnItsWay<St, WIDE, THREADS> tp, pp;
    StepsOnTheirWay<THREADS> sp;
    Sixteen<E> op;
    auto fetch = [&](int64_t n) {
        const int64_t t0 = n * C;
        const int rows = int(S.T - t0 < C ? S.T - t0 : C);
        kp.load(k0 + t0 * S.kt, S.kt, rows, S.K);
        qp.load(q0 + t0 * S.qt, S.qt, rows, S.K);
#pragma unroll
        for (int j = 0; j < In8::COUNT; j++) {
            kr[j] = rec[n].steps.rk[In8::row(j)];
            qr[j] = rec[n].steps.rq[In8::row(j)];
        }
        tp.load(rec[n].inv);
        pp.load(rec[n].pair);
        sp.load(rec[n].steps);
        op.load(o0 + t0 * S.ot, S.ot, rows);
    };
    const auto four = [&](const float* p, int it) { return *reinterpret_cast<const f4*>(p + 16 * it + 4 * grp); };

    In8::clear(Kt, S.K);
    In8::clear(Qt, S.K);
    fetch(S.chunks - 1);
    for (int64_t n = S.chunks - 1; n >= 0; n--) {
        __syncthreads();                   // the chunk after has been used
#pragma unroll
        for (int j = 0; j < In8::COUNT; j++) {
            kp.put(Kt, j, length_up<St>(kr[j]), S.K);
            qp.put(Qt, j, length_up<St>(qr[j]), S.K);
        }
        tp.put(Tt);
        pp.put(Pt);
        sp.put(st);
        const int64_t t0 = n * C;
        f4 o[4];
#pragma unroll
        for (int it = 0; it < 4; it++) {
            o[it] = op.four(it, on);
#pragma unroll
            for (int r = 0; r < 4; r++) if (t0 + 16 * it + 4 * grp + r >= S.T) o[it][r] = 0.0f;
        }
        __syncthreads();
        if (n) fetch(n - 1);
        const int64_t row = (bg * S.chunks + n) * S.vp + col;
        const Scale ss = scale_of<St>(over_column(largest(s))), os = scale_of<St>(over_column(largest(o)));
        Frag<St, WIDE> sf[KB];
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
            sf[kb] = frag_of<St, WIDE>(s[2 * kb], s[2 * kb + 1], ss.up);
            if (held) leave(walked.states + row * DK + 32 * kb + 8 * grp, sf[kb]);
        }
        // dU = l K dS + P^T dO
        Frag<St, 1> of[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) of[kb] = frag_of<St, 1>(o[2 * kb], o[2 * kb + 1], os.up);       // (these are a tensor's elements: nothing is rounded off)
        const float dp = os.down * (1.0f / SQUARE<St>);
        f4 u[4];
#pragma unroll
        for (int it = 0; it < 4; it++) {
            f4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
#pragma unroll
            for (int kb = 0; kb < KB; kb++) mma(x, Kt.rows(16 * it, kb), sf[kb]);
#pragma unroll
            for (int kb = it / 2; kb < 2; kb++) mma(y, Pt.cols(16 * it, kb), of[kb]);
            const f4 ls = four(st.l, it);
#pragma unroll
            for (int r = 0; r < 4; r++) u[it][r] = fmaf(dp, y[r], ls[r] == 0.0f ? 0.0f : ls[r] * (ss.down * x[r]));
        }
        // dR = T^T dU
        const Scale us = scale_of<St>(over_column(largest(u)));
        Frag<St, WIDE> uf[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) uf[kb] = frag_of<St, WIDE>(u[2 * kb], u[2 * kb + 1], us.up);
        const float du = us.down * (1.0f / SQUARE<St>);
        f4 d[4];
#pragma unroll
        for (int it = 0; it < 4; it++) {
            d[it] = f4{0, 0, 0, 0};
#pragma unroll
            for (int kb = it / 2; kb < 2; kb++) mma(d[it], Tt.cols(16 * it, kb), uf[kb]);
            d[it] *= du;
        }
        const Scale ds = scale_of<St>(over_column(largest(d)));
        E* to = d_value + ((b * S.T + t0) * S.G + g) * S.V + col;
        f4 x[4], y[4];
#pragma unroll
        for (int it = 0; it < 4; it++) {
            const f4 bs = four(st.b, it), bd = bs * d[it];
            x[it] = four(st.q, it) * o[it];
            y[it] = -four(st.x, it) * bd;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int i = 16 * it + 4 * grp + r;
                if (on && t0 + i < S.T) to[int64_t(i) * S.G * S.V] = E(bd[r]);
            }
        }
        const Scale xs = scale_of<St>(over_column(fmaxf(largest(x), largest(y))));
        Frag<St, WIDE> xf[2], yf[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            if (held) leave(walked.steps + row * C + 32 * kb + 8 * grp, frag_of<St, 1>(d[2 * kb], d[2 * kb + 1], ds.up));
            xf[kb] = frag_of<St, WIDE>(x[2 * kb], x[2 * kb + 1], xs.up);
            yf[kb] = frag_of<St, WIDE>(y[2 * kb], y[2 * kb + 1], xs.up);
        }
        if (held && grp == 0) {
            float* scales = walked.scales + (bg * S.chunks + n) * 3 * S.vp + col;
            scales[0] = ss.down;
            scales[S.vp] = ds.down;
            scales[2 * S.vp] = os.down;
        }
        const float end = st.end;
#pragma unroll
        for (int k = 0; k < ND; k++) {
            f4 z = {0, 0, 0, 0};
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                mma(z, Qt.cols(16 * k, kb), xf[kb]);
                mma(z, Kt.cols(16 * k, kb), yf[kb]);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) s[k][r] = fmaf(xs.down, z[r], end == 0.0f ? 0.0f : end * s[k][r]);
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
//
// Five products are summed over columns of values, whose operands have a scale for each column. The two scales of a column go to the
// left operand, over the largest of them: what they push below float16's numbers is that far below the sum's largest terms.

constexpr int BLOCK_V = 32, PRODUCTS = 5;

__device__ inline float row16(float x) {   // a sum over the 16 lanes that have a row's columns
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) x += __shfl_xor(x, d, WAVE);
    return x;
}
__device__ inline int exponent(float x) { return int(__float_as_uint(x) >> 23) - 127; }

template <typename E, int DK>
__global__ __launch_bounds__(BLOCK) void gradient_kernel(const E* __restrict__ query, const E* __restrict__ key, const E* __restrict__ gate, const E* __restrict__ write,
                                                         const E* __restrict__ d_out, Shape S, const Chunk<typename Rep<E>::S>* __restrict__ records,
                                                         const Kept<typename Rep<E>::S> kept, const Kept<typename Rep<E>::S> walked, E* __restrict__ d_query,
                                                         E* __restrict__ d_key, E* __restrict__ d_gate, E* __restrict__ d_write) {
    using St = typename Rep<E>::S;
    constexpr bool HALF = sizeof(St) == 2;
    constexpr int ND = DK / 16, KB = DK / 32, PER = DK / 8;
    using In = Tile<St, C, DK>;
    using Ot = Tile<St, C, BLOCK_V>;
    using Sv = Tile<St, BLOCK_V, DK>;
    using Uv = Tile<St, BLOCK_V, C>;
    using Square = Tile<St, C, C>;
    using In8 = Rows<E, DK, BLOCK>;
    constexpr int STAGED = Ot::SIZE + 2 * Sv::SIZE + 2 * Uv::SIZE, MORE = STAGED > 3 * Square::SIZE ? STAGED : 3 * Square::SIZE;
    __shared__ alignas(16) St lds[2 * In::SIZE + MORE];
    __shared__ alignas(16) Steps st;
    __shared__ alignas(16) St factors[PRODUCTS][BLOCK_V];
    __shared__ float rows[C], columns[WAVES][C], left[C], whole[WAVES], writes[C];
    __shared__ int tops[WAVES][PRODUCTS];
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
    // products of E and F with keys and queries, over numbers of values each
    const int many = HALF ? 32 - __builtin_clz(S.V) : 0;
    const float few = __uint_as_float((127 - many) << 23);
    {
        In8 q, k;
        float qr[In8::COUNT], kr[In8::COUNT];
        const Steps& first = records[(b * S.G + h * share) * S.chunks + chunk].steps;
        q.load(query + b * S.qb + t0 * S.qt + h * S.qh, S.qt, steps, S.K);
        k.load(key + b * S.kb + t0 * S.kt + h * S.kh, S.kt, steps, S.K);
#pragma unroll
        for (int j = 0; j < In8::COUNT; j++) {
            kr[j] = first.rk[In8::row(j)];
            qr[j] = first.rq[In8::row(j)];
        }
        In8::clear(Qt, S.K);
        In8::clear(Kt, S.K);
#pragma unroll
        for (int j = 0; j < In8::COUNT; j++) {
            q.put(Qt, j, length_up<St>(qr[j]), S.K);
            k.put(Kt, j, length_up<St>(kr[j]), S.K);
        }
    }
    const f4 zero = {0, 0, 0, 0};
    f4 tq[ND], tk[ND];                     // the gradients of the query and the key of length 1, over the value heads so far
#pragma unroll
    for (int n = 0; n < ND; n++) tq[n] = tk[n] = zero;

    for (int j = 0; j < share; j++) {
        const int g = h * share + j;
        const int64_t at = (b * S.G + g) * S.chunks + chunk;
        const E* o0 = d_out + b * S.ob + t0 * S.ot + g * S.og;
        const St *s0 = kept.states + at * S.vp * DK, *s1 = walked.states + at * S.vp * DK, *u0 = kept.steps + at * S.vp * C, *r0 = walked.steps + at * S.vp * C;
        const float *f0 = kept.scales + at * 3 * S.vp, *f1 = walked.scales + at * 3 * S.vp;    // of S, U and of dS, dR, dO
        const auto left_scale = [&](int p, int c) { return p == 2 ? f0[S.vp + c] : p == 0 || p == 3 ? f1[2 * S.vp + c] : f1[S.vp + c]; };
        const auto right_scale = [&](int p, int c) { return p < 2 ? f0[c] : p == 2 ? f1[c] : f0[S.vp + c]; };
        if constexpr (HALF) {              // the largest of the columns' scales, by product: dO S, dR S, U dS, dO U, dR U
            int top[PRODUCTS];
#pragma unroll
            for (int p = 0; p < PRODUCTS; p++) top[p] = -1000;
            for (int c = tid; c < S.vp; c += BLOCK) {
                const int es = exponent(f0[c]), eu = exponent(f0[S.vp + c]), ed = exponent(f1[c]), er = exponent(f1[S.vp + c]), eo = exponent(f1[2 * S.vp + c]);
                top[0] = max(top[0], eo + es);
                top[1] = max(top[1], er + es);
                top[2] = max(top[2], eu + ed);
                top[3] = max(top[3], eo + eu);
                top[4] = max(top[4], er + eu);
            }
#pragma unroll
            for (int p = 0; p < PRODUCTS; p++) {
#pragma unroll
                for (int d = WAVE / 2; d; d >>= 1) top[p] = max(top[p], __shfl_xor(top[p], d, WAVE));
                if (l == 0) tops[wave][p] = top[p];
            }
        }
        f4 aq[ND], from[ND], to[ND], dp[WAVES], da[WAVES];
#pragma unroll
        for (int n = 0; n < ND; n++) aq[n] = from[n] = to[n] = zero;
#pragma unroll
        for (int n = 0; n < WAVES; n++) dp[n] = da[n] = zero;
        float both = 0.0f;                 // of state and gradient, summed over all elements
        constexpr int SP = BLOCK_V * PER / BLOCK ? BLOCK_V * PER / BLOCK : 1;
        pack<E, 8> op;
        pack<float, 8> os;
        pack<St, 8> s0p[SP], s1p[SP], up, rp;
        float sd[SP], lf, rf;
        // (columns behind the last are read as the last one and put as 0; d_out's last eight one by one where V is no multiple of 8)
        const int oc = tid % 4 * 8, orow = tid / 4, urow = tid / 8, ucol = tid % 8 * 8;
        const E* orow0 = o0 + int64_t(orow < steps ? orow : steps - 1) * S.ot;
        const auto last = [&](int c) { return c < S.vp ? c : S.vp - 1; };
        auto fetch = [&](int v0) {
            if (S.V % 8 == 0) {
                op = pack<E, 8>::load(orow0 + (v0 + oc < S.V ? v0 + oc : S.V - 8));
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) op.v[e] = orow0[v0 + oc + e < S.V ? v0 + oc + e : S.V - 1];
            }
            if constexpr (HALF) {
                os = pack<float, 8>::load(f1 + 2 * S.vp + (v0 + oc < S.vp ? v0 + oc : S.vp - 8));
                lf = left_scale(tid / BLOCK_V < PRODUCTS ? tid / BLOCK_V : 0, last(v0 + tid % BLOCK_V));
                rf = right_scale(tid / BLOCK_V < PRODUCTS ? tid / BLOCK_V : 0, last(v0 + tid % BLOCK_V));
            }
            up = pack<St, 8>::load(u0 + int64_t(last(v0 + urow)) * C + ucol);
            rp = pack<St, 8>::load(r0 + int64_t(last(v0 + urow)) * C + ucol);
#pragma unroll
            for (int k = 0; k < SP; k++) {
                const int p = tid + k * BLOCK, c = last(v0 + p / PER);
                s0p[k] = pack<St, 8>::load(s0 + int64_t(c) * DK + p % PER * 8);
                s1p[k] = pack<St, 8>::load(s1 + int64_t(c) * DK + p % PER * 8);
                if constexpr (HALF) sd[k] = f0[c] * f1[c];
                else sd[k] = 1.0f;
            }
        };
        fetch(0);
        for (int v0 = 0; v0 < S.vp; v0 += BLOCK_V) {
            __syncthreads();               // what lies there has been used
            {
                St x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float d = v0 + oc + e < S.V ? float(op.v[e]) : 0.0f;
                    x[e] = St(HALF ? d * __uint_as_float((254u << 23) - __float_as_uint(os.v[e])) : d);    // (over a power of two)
                }
                Od.put(orow, oc, x);
            }
            if constexpr (HALF) if (tid < PRODUCTS * BLOCK_V) {
                const int p = tid / BLOCK_V, c = tid % BLOCK_V;
                const int top = max(max(tops[0][p], tops[1][p]), max(tops[2][p], tops[3][p]));
                const int e = exponent(lf) + exponent(rf) - top;   // 0 at most
                factors[p][place(c)] = v0 + c < S.vp && e > -25 ? St(__uint_as_float((127 + e) << 23)) : St(0.0f);
            }
            const pack<St, 8> none = {};
            Us.put_places(urow, ucol, v0 + urow < S.vp ? up : none);
            Rs.put_places(urow, ucol, v0 + urow < S.vp ? rp : none);
#pragma unroll
            for (int k = 0; k < SP; k++) {
                const int p = tid + k * BLOCK;
                if (p < BLOCK_V * PER) {
                    const bool on = v0 + p / PER < S.vp;
                    S0.put_places(p / PER, p % PER * 8, on ? s0p[k] : none);
                    S1.put_places(p / PER, p % PER * 8, on ? s1p[k] : none);
                    float x = 0.0f;
#pragma unroll
                    for (int c = 0; c < 8; c++) x = fmaf(float(s0p[k].v[c]), float(s1p[k].v[c]), x);
                    if (on) both = fmaf(x, sd[k], both);
                }
            }
            if (v0 == 0) {                 // the steps' record with the first block
                const float* p = reinterpret_cast<const float*>(&records[at].steps);
                for (int k = tid; k < int(sizeof(Steps) / 4); k += BLOCK) reinterpret_cast<float*>(&st)[k] = p[k];
            }
            __syncthreads();
            if (v0 + BLOCK_V < S.vp) fetch(v0 + BLOCK_V);
            const auto scaled = [&](auto f, int p) {
                if constexpr (HALF) f.p[0] *= *reinterpret_cast<const h8*>(&factors[p][8 * grp]);
                return f;
            };
            const auto of = Od.rows(band, 0);
            const auto rf = Rs.cols(band, 0), uf = Us.cols(band, 0);
            const auto of0 = scaled(of, 0), rf1 = scaled(rf, 1), uf2 = scaled(uf, 2), of3 = scaled(of, 3), rf4 = scaled(rf, 4);
#pragma unroll
            for (int n = 0; n < ND; n++) {
                const auto sf = S0.cols(16 * n, 0);
                mma(aq[n], of0, sf);
                mma(from[n], rf1, sf);
                mma(to[n], uf2, S1.cols(16 * n, 0));
            }
#pragma unroll
            for (int n = 0; n < WAVES; n++) if (n <= wave) {
                const auto un = Us.cols(16 * n, 0);
                mma(dp[n], of3, un);
                mma(da[n], rf4, un);
            }
        }
        int top[PRODUCTS];
#pragma unroll
        for (int p = 0; p < PRODUCTS; p++) top[p] = HALF ? max(max(tops[0][p], tops[1][p]), max(tops[2][p], tops[3][p])) : 0;
        const uint64_t cuts = uint64_t(st.cut[1]) << 32 | st.cut[0];
        // what a step has of the state before the chunk and leaves after it, and its row's sums
        float bi[4], rowsum[4], rki[4], rqi[4];
        const float last_hi = st.hi[C - 1], last_lo = st.lo[C - 1];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = band + 4 * grp + r;
            const float gi = since(cuts, i) >= 0 ? 0.0f : expf(st.hi[i]);
            const float li = i < since(cuts, C - 1) ? 0.0f : expf((last_hi - st.hi[i]) + (last_lo - st.lo[i]));
            bi[r] = st.b[i];
            rki[r] = length_rest<St>(st.rk[i]);
            rqi[r] = length_rest<St>(st.rq[i]);
            float dq = 0.0f, df = 0.0f, dt = 0.0f;
#pragma unroll
            for (int n = 0; n < ND; n++) {
                const float x = gi == 0.0f ? 0.0f : gi * ldexpf(aq[n][r], top[0]), y = gi == 0.0f ? 0.0f : -bi[r] * gi * ldexpf(from[n][r], top[1]);
                const float z = li == 0.0f ? 0.0f : li * ldexpf(to[n][r], top[2]);
                const float q = float(Qt.get(i, 16 * n + m)), k = float(Kt.get(i, 16 * n + m));
                dq = fmaf(q, x, dq);
                df = fmaf(k, y, df);
                dt = fmaf(k, z, dt);
                tq[n][r] += x;
                tk[n][r] += y + z;
            }
            rowsum[r] = rqi[r] * dq + rki[r] * df;
            dt = row16(dt);
            if (m == 0) left[i] = rki[r] * dt;
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
            const float rk = length_rest<St>(st.rk[c]), hi = st.hi[c], lo = st.lo[c];
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
                        const float pair = ldexpf(e * rqi[r] * rk * qk[n][r], top[3]) + ldexpf(f * rki[r] * rk * kk[n][r], top[4]);
                        rowsum[r] += pair;
                        column += pair;
                    } else {
                        writes[i] = ldexpf(da[n][r], top[4]);
                    }
                }
                // (numbers up to 2^28 V, of factors up to 2^14: V 2^14 of them, and lengths, are taken out)
                constexpr float FIT = HALF ? 0x1p-15f * LONG<St> : 1.0f;
                e *= few * FIT;
                f *= few * FIT;
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
        constexpr int OUT = HALF ? 15 - 6 : 0;             // (what FIT took out)
        static_assert(!HALF || LONG<St> == 64.0f, "the exponent of LONG");
#pragma unroll
        for (int n = 0; n < ND; n++) {
            f4 x = zero, y = zero, z = zero;
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                const auto kn = Kt.cols(16 * n, kb);
                mma(x, Ek.rows(band, kb), kn);
                mma(y, Eq.cols(band, kb), Qt.cols(16 * n, kb));
                mma(z, Ff.rows(band, kb), kn);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                tq[n][r] += ldexpf(x[r], top[3] + many + OUT);
                tk[n][r] += ldexpf(y[r], top[3] + many + OUT) + ldexpf(z[r], top[4] + many + OUT);
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
        const float rk = st.rk[i], rq = st.rq[i], rkr = length_rest<St>(rk), rqr = length_rest<St>(rq);
        float q[ND], k[ND], dq = 0.0f, dk = 0.0f;
#pragma unroll
        for (int n = 0; n < ND; n++) {
            q[n] = float(Qt.get(i, 16 * n + m)) * rqr;
            k[n] = float(Kt.get(i, 16 * n + m)) * rkr;
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
