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
//
// What bounds it. bfloat16, 8 sequences of 8,192 steps, 8 heads of 128 x 128: walk_kernel 653 us, as state_kernel; gradient_kernel 816, 57,000 cycles
// a chunk on a CU that has room for one (155 KB of LDS, 256 registers a lane): 21,000 of them issue vector operations on each SIMD, 7,400 its matrix unit is
// busy, the rest are waits for the first block, LDS and barriers.
#include "pv_delta.h"

using namespace pvd;

namespace {

// ---- walk_kernel: a workgroup of W waves for 16 W columns of a state's gradient, and a wave more that brings chunks to LDS

// MAP: the first walk of a sequence in pieces, each from a gradient of zero behind it; nothing is left but the gradient before it.
template <typename E, int DK, int W, bool MAP>
__global__ __launch_bounds__((W + 1) * WAVE) __attribute__((amdgpu_waves_per_eu(1, 2))) void walk_kernel(
    const E* __restrict__ d_out, const float* __restrict__ d_last, Shape S, const char* __restrict__ records, const char* __restrict__ images, E* __restrict__ d_value,
    float* __restrict__ d_state, Kept<Rep<E>, DK> walked, Pieces pieces, Joins joins) {
    using St = Rep<E>;
    using Ke = Kept<St, DK>;
    constexpr int WIDE = wide_of<St>, ND = DK / 16, KB = DK / 32;
    using In = Tile<St, C, DK>;
    using Square = Tile<St, C, C, WIDE>;
    using Re = Record<St>;
    constexpr int BUFFERS = sizeof(St) == 2 ? 2 : 1, IN = IMAGE<St, DK>, BUFFER = IN + Re::STRIDE;
    __shared__ alignas(1024) char lds[BUFFERS * BUFFER];
    const int tid = threadIdx.x, wave = tid / WAVE, l = tid % WAVE, grp = l / 16, m = l % 16;
    const int groups = (S.vp / 16 + W - 1) / W;
    const auto [piece, group] = part_of(blockIdx.x, S.B * S.G * pieces.count, groups);
    const int col = (group * W + wave) * 16 + m;
    const int64_t bg = piece / pieces.count, b = bg / S.G, first = piece % pieces.count * pieces.chunks;
    const int64_t behind = first + pieces.chunks < S.chunks ? first + pieces.chunks : S.chunks;
    const int g = int(bg % S.G), h = shared(S, g);
    const bool on = col < S.V;
    const E* o0 = d_out + b * S.ob + g * S.og;
    const char *rec0 = records + bg * S.chunks * Re::STRIDE, *in0 = images + (b * S.H + h) * S.chunks * IN;
    const int vt = S.G * S.V;              // steps of d_value
    const uint32_t out_at = Sixteen<E>::first(S.ot, col, on), value_at = Sixteen<E>::first(vt, col, on);
    const uint32_t state_at = Ke::state_at(col, S.vp) + 8 * grp * sizeof(St), step_at = Ke::step_at(col, S.vp) + 8 * grp * sizeof(St);

    f4 s[ND];
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 16 * n + 4 * grp + r;
            if constexpr (MAP) s[n][r] = 0.0f;
            else if (behind < S.chunks) s[n][r] = col < S.vp ? joins.starts[(piece * S.vp + col) * DK + d] : 0.0f;
            else s[n][r] = d_last && on && d < S.K ? d_last[(bg * S.K + d) * S.V + col] : 0.0f;
        }
    const auto rows_of = [&](int64_t n) { return int(S.T - n * C < C ? S.T - n * C : C); };
    if (wave == W) {
        for (int64_t n = behind - 1; n >= first; n--) {
            if (n < behind - 1 && BUFFERS == 1) __syncthreads();       // the chunk after has been used
            char* to = lds + (BUFFERS == 2 ? int(n & 1) * BUFFER : 0);
            bring<1>(in0 + n * IN, to, 2 * In::SIZE * int(sizeof(St)), 0);
            bring<1>(rec0 + n * Re::STRIDE, to + IN, Re::ALL, 0);
            arrived<0>();
            __syncthreads();               // the chunk is there (and of two, the one after has been used)
        }
        return;
    }
    Sixteen<E> op;
    op.load(rows_at(o0 + (behind - 1) * C * S.ot, S.ot, rows_of(behind - 1), S.V), S.ot, out_at);
    for (int64_t n = behind - 1; n >= first; n--) {
        if (n < behind - 1 && BUFFERS == 1) __syncthreads();
        __syncthreads();
        char* here = lds + (BUFFERS == 2 ? int(n & 1) * BUFFER : 0);
        const In Kt{reinterpret_cast<St*>(here)}, Qt{reinterpret_cast<St*>(here) + In::SIZE};
        const Re& re = *reinterpret_cast<const Re*>(here + IN);
        const Steps& st = re.steps;
        const Square Tt{const_cast<St*>(&re.inv[0][0][0])}, Pt{const_cast<St*>(&re.pair[0][0][0])};
        const auto four = [&](const float* p, int it) { return *reinterpret_cast<const f4*>(p + 16 * it + 4 * grp); };
        const int rows = rows_of(n);
        const uint64_t cuts = uint64_t(st.cut[1]) << 32 | st.cut[0];
        f4 o[4];
#pragma unroll
        for (int it = 0; it < 4; it++) o[it] = op.four(it);
        uint64_t odd = uint64_t(st.odd[1] | st.odd_query[1]) << 32 | st.odd[0] | st.odd_query[0];
        const bool some = __builtin_amdgcn_readfirstlane(uint32_t(odd >> 32) | uint32_t(odd)) || __any(not_finite(o) != 0.0f);
        if (some) odd |= taken_out(o) & (~0ull >> (C - rows));
        bool lost = false;                 // the gradient after a chunk in which some step drops the state is not finite
        by_cut(cuts, [&](auto cut) {
            if constexpr (decltype(cut)::value) {
                lost = over_column(not_finite(s)) != 0.0f;
#pragma unroll
                for (int k = 0; k < ND; k++)
#pragma unroll
                    for (int r = 0; r < 4; r++) s[k][r] = lost ? 0.0f : s[k][r];
            }
        });
        if (n > first) op.load(rows_at(o0 + (n - 1) * C * S.ot, S.ot, rows_of(n - 1), S.V), S.ot, out_at);
        const int64_t at = (bg * S.chunks + n) * S.vp;     // of the chunk in what is left over
        const Buffer blocks(walked.blocks + at / COLS * Ke::BLOCK, int64_t(S.vp / COLS) * Ke::BLOCK * int(sizeof(St)));
        // operands of a stage's products are loaded while the stage before runs
        Frag<St, 1> ka[KB][4], of[2];
        Frag<St, WIDE> pa[2][4], ta[2][4], sf[KB];
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int it = 0; it < 2 * kb + 2; it++) pa[kb][it] = Pt.cols(16 * it, kb);
#pragma unroll
        for (int kb = 0; kb < KB; kb++)
#pragma unroll
            for (int it = 0; it < 4; it++) ka[kb][it] = Kt.rows(16 * it, kb);
        fence();
        const Scale ss = scale_of<St>(over_column(largest(s))), os = scale_of<St>(over_column(largest(o)));
#pragma unroll
        for (int kb = 0; kb < 2; kb++) of[kb] = frag_of<St, 1>(o[2 * kb], o[2 * kb + 1], os.up);       // (these are a tensor's elements: nothing is rounded off)
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
            sf[kb] = frag_of<St, WIDE>(s[2 * kb], s[2 * kb + 1], ss.up);
            if constexpr (!MAP) leave(blocks, state_at + 32 * kb * sizeof(St), sf[kb], Ke::STATES);
        }
        // dU = l K dS + P^T dO
        const float dp = os.down * (1.0f / SQUARE<St>);
        f4 u[4], w[4];
#pragma unroll
        for (int it = 0; it < 4; it++) u[it] = w[it] = f4{0, 0, 0, 0};
        mma_first(w, pa[0], of[0]);
        mma_all(w, pa[1], of[1]);
        fence();
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int it = 0; it < 2 * kb + 2; it++) ta[kb][it] = Tt.cols(16 * it, kb);
#pragma unroll
        for (int kb = 0; kb < KB; kb++) mma_all(u, ka[kb], sf[kb]);
        by_cut(cuts, [&](auto cut) {
#pragma unroll
            for (int it = 0; it < 4; it++) u[it] = part_of_it<decltype(cut)::value>(four(st.l, it) * ss.down, u[it]) + dp * w[it];
        });
        // dR = T^T dU
        const Scale us = scale_of<St>(over_column(largest(u)));
        Frag<St, WIDE> uf[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) uf[kb] = frag_of<St, WIDE>(u[2 * kb], u[2 * kb + 1], us.up);
        const float du = us.down * (1.0f / SQUARE<St>);
        fence();
        Frag<St, 1> kc[2][ND], qc[2][ND];
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int k = 0; k < ND; k++) {
                qc[kb][k] = Qt.cols(16 * k, kb);
                kc[kb][k] = Kt.cols(16 * k, kb);
            }
        f4 d[4];
#pragma unroll
        for (int it = 0; it < 4; it++) d[it] = f4{0, 0, 0, 0};
        mma_first(d, ta[0], uf[0]);
        mma_all(d, ta[1], uf[1]);
        const Scale ds = scale_of<St>(over_column(largest(d)) * du);
        const Buffer to = rows_at(d_value + ((b * S.T + n * C) * S.G + g) * S.V, vt, rows, S.V);
        f4 x[4], y[4];
#pragma unroll
        for (int it = 0; it < 4; it++) {
            const f4 bs = four(st.b, it) * du;
            x[it] = four(st.q, it) * o[it];
            y[it] = four(st.x, it) * d[it] * -du;
#pragma unroll
            for (int r = 0; r < 4; r++) if constexpr (!MAP) Sixteen<E>::store(to, vt, value_at, 4 * it + r, bs[r] * d[it][r]);
        }
        // (q and x are 2 / LONG at most)
        const Scale xs = scale_of<St>(over_column(fmaxf(largest(x), largest(y))));
        Frag<St, WIDE> xf[2], yf[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            if constexpr (!MAP) leave(blocks, step_at + 32 * kb * sizeof(St), frag_of<St, WIDE>(d[2 * kb], d[2 * kb + 1], sizeof(St) == 2 ? du * ds.up : 1.0f), Ke::STEPS);
            xf[kb] = frag_of<St, WIDE>(x[2 * kb], x[2 * kb + 1], xs.up);
            yf[kb] = frag_of<St, WIDE>(y[2 * kb], y[2 * kb + 1], xs.up);
        }
        const Buffer scales(walked.scales + 3 * at, 3 * int64_t(S.vp) * 4);
        const uint32_t scale_at = grp == 0 && col < S.vp ? col * 4 : NOWHERE;
        if constexpr (!MAP) {
            scales.store(ss.down, scale_at);
            scales.store(ds.down, scale_at, S.vp * 4);
            scales.store(os.down, scale_at, 2 * S.vp * 4);
        }
        fence();
        const float end = st.end;
        f4 z[ND];
#pragma unroll
        for (int k = 0; k < ND; k++) z[k] = f4{0, 0, 0, 0};
#pragma unroll
        for (int kb = 0; kb < 2; kb++) mma_all(z, qc[kb], xf[kb]);
#pragma unroll
        for (int kb = 0; kb < 2; kb++) mma_all(z, kc[kb], yf[kb]);
        by_cut(cuts, [&](auto cut) {
#pragma unroll
            for (int k = 0; k < ND; k++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[k][r] = fmaf(xs.down, z[k][r], part_of_it<decltype(cut)::value>(end, s[k][r]));
        });
        if (some || __any(lost)) {         // (the gradients take from what is left which steps are NaN; their own products are by steps and heads)
            const int first4 = thread() % WAVE / 16 * 4;
            const auto spoils = [&](int i) { return reached_back(odd, cuts, i) || (lost && i >= since(cuts, C - 1)); };
            if constexpr (!MAP) {
#pragma unroll
                for (int it = 0; it < 4; it++)
#pragma unroll
                    for (int r = 0; r < 4; r++) Sixteen<E>::store(to, vt, spoils(16 * it + first4 + r) ? value_at : NOWHERE, 4 * it + r, NAN);
#pragma unroll
                for (int kb = 0; kb < 2; kb++) spoil<St>(blocks, step_at + 32 * kb * sizeof(St), 32 * kb + first4, spoils);
#pragma unroll
                for (int kb = 0; kb < KB; kb++) spoil<St>(blocks, state_at + 32 * kb * sizeof(St), 0, [&](int) { return lost; });
            }
            if (odd & (cuts ? (cuts & -cuts) - 1 : ~0ull))
#pragma unroll
                for (int k = 0; k < ND; k++) s[k] = f4{NAN, NAN, NAN, NAN};
        }
    }
    if constexpr (MAP) {
        if (col < S.vp) {
            float* to = joins.ends + (piece * (S.vp + DK) + col) * DK + 4 * grp;
#pragma unroll
            for (int n = 0; n < ND; n++) *reinterpret_cast<f4*>(to + 16 * n) = s[n];
        }
        return;
    }
    if (!d_state || first) return;
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 16 * n + 4 * grp + r;
            if (on && d < S.K) d_state[(bg * S.K + d) * S.V + col] = s[n][r];
        }
}

// ---- gradient_kernel: a workgroup of eight waves for each chunk of each query and key head. A wave has 16 steps' rows of every product
// and half of its columns; columns of values are summed over in blocks of 32, which come to LDS while the block before is used where
// two have room.
//
// Five products are summed over columns of values, whose operands have a scale for each column. The two scales of a column go to the
// left operand, over the largest of them: what they push below float16's numbers is that far below the sum's largest terms.

constexpr int BANDS = 4, HALVES = 2, MANY = BANDS * HALVES * WAVE, PRODUCTS = 5;

// x at place `at` of a tile's row, in parts
template <typename T> __device__ inline void put_parts(const T& tile, int row, int at, float x) {
    using S = typename T::S;
    if constexpr (sizeof(S) == 2) asm("" : "+v"(x));       // (as in frag_of)
    S* to = tile.p + row * T::ROW + at;
#pragma unroll
    for (int w = 0; w < T::SIZE / T::PLANE; w++) {
        to[w * T::PLANE] = S(x);
        x -= float(S(x));
    }
}

__device__ inline int exponent(float x) { return int(__float_as_uint(x) >> 23) - 127; }

template <typename E, int DK>
__global__ __launch_bounds__(MANY) __attribute__((amdgpu_waves_per_eu(2, 2))) void gradient_kernel(const E* __restrict__ gate, const E* __restrict__ write, const E* __restrict__ d_out, Shape S,
                                                        const char* __restrict__ records, const char* __restrict__ images, const Kept<Rep<E>, DK> kept,
                                                        const Kept<Rep<E>, DK> walked, E* __restrict__ d_query, E* __restrict__ d_key,
                                                        E* __restrict__ d_gate, E* __restrict__ d_write) {
    using St = Rep<E>;
    using Ke = Kept<St, DK>;
    using Re = Record<St>;
    constexpr bool HALF = sizeof(St) == 2;
    constexpr int WIDE = wide_of<St>, ND = DK / 16 / HALVES, KB = DK / 32, WAVES = MANY / WAVE, UNIT = 16 / int(sizeof(St));
    using In = Tile<St, C, DK>;
    using Ot = Tile<St, C, COLS>;
    using Sv = Tile<St, COLS, DK, WIDE>;
    using Uv = Tile<St, COLS, C, WIDE>;
    using Square = Tile<St, C, C, WIDE>;
    static_assert(Sv::SIZE + Uv::SIZE == Ke::BLOCK, "blocks lie in LDS as they are kept");
    constexpr int BUFFERS = HALF ? 2 : 1, IN = IMAGE<St, DK>, BLOCK = Ke::BLOCK * int(sizeof(St)), BUFFER = 2 * BLOCK + Ot::SIZE * int(sizeof(St));
    constexpr int MORE = BUFFERS * BUFFER > 3 * Square::SIZE * int(sizeof(St)) ? BUFFERS * BUFFER : 3 * Square::SIZE * int(sizeof(St));
    __shared__ alignas(1024) char lds[IN + MORE];
    __shared__ alignas(16) Steps st;
    __shared__ alignas(16) St factors[2][PRODUCTS][COLS];
    __shared__ float rows[HALVES][C], columns[BANDS][C], left[HALVES][C], whole[WAVES], writes[C], dots[2][HALVES][C];
    __shared__ int tops[WAVES][PRODUCTS];
    __shared__ double gates[2][C];
    const In Kt{reinterpret_cast<St*>(lds)}, Qt{reinterpret_cast<St*>(lds) + In::SIZE};
    St* const more = reinterpret_cast<St*>(lds + IN);
    const Square Ek{more}, Eq{more + Square::SIZE}, Ff{more + 2 * Square::SIZE};       // (once the blocks of values have been used)
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), half = wave / BANDS,
              own = half ? BANDS - 1 - wave % BANDS : wave % BANDS,    // (the two of a SIMD have near as much up to the diagonal as any other two)
              band = 16 * own, d0 = half * DK / 2;
    const int64_t chunk = blockIdx.x % S.chunks, bh = blockIdx.x / S.chunks;
    const int64_t b = bh / S.H, t0 = chunk * C;
    const int h = int(bh % S.H), share = S.G / S.H, steps = int(S.T - t0 < C ? S.T - t0 : C);
    // products of E and F with keys and queries, over numbers of values each
    const int many = HALF ? 32 - __builtin_clz(S.V) : 0;
    const float few = __uint_as_float((127 - many) << 23);
    const f4 zero = {0, 0, 0, 0};
    f4 tq[ND], tk[ND];                     // the gradients of the query and the key of length 1, over the value heads so far
#pragma unroll
    for (int n = 0; n < ND; n++) tq[n] = tk[n] = zero;

    for (int j = 0; j < share; j++) {
        const int g = h * share + j;
        const int64_t at = (b * S.G + g) * S.chunks + chunk;
        const E* o0 = d_out + b * S.ob + t0 * S.ot + g * S.og;
        const St *b0 = kept.blocks + at * (S.vp / COLS) * Ke::BLOCK, *b1 = walked.blocks + at * (S.vp / COLS) * Ke::BLOCK;
        const float *f0 = kept.scales + at * 3 * S.vp, *f1 = walked.scales + at * 3 * S.vp;    // of S, U and of dS, dR, dO
        f4 aq[ND], from[ND], to[ND], dp[2], da[2];     // (of 16 x 16 up to the diagonal a wave has those at columns half, half + 2)
#pragma unroll
        for (int n = 0; n < ND; n++) aq[n] = from[n] = to[n] = zero;
        dp[0] = dp[1] = da[0] = da[1] = zero;
        float both = 0.0f;                 // of state and gradient, summed over all elements
        // (kept as they come: 16 bits made 32 of are waited for at once where their loads are behind a branch)
        std::conditional_t<sizeof(E) == 2, uint16_t, uint32_t> op[4];
        f4 os = {1.0f, 1.0f, 1.0f, 1.0f};
        float lf = 1.0f, rf = 1.0f;
        const float *lp = f1, *rp = f0;    // of the lane's product and column
        int most = 0;                      // the largest of that product's scales
        if constexpr (HALF) {
            const int tid = thread(), product = tid / COLS < PRODUCTS ? tid / COLS : 0, column = tid % COLS;
            lp = (product == 2 ? f0 + S.vp : product == 0 || product == 3 ? f1 + 2 * S.vp : f1 + S.vp) + column;
            rp = (product < 2 ? f0 : product == 2 ? f1 : f0 + S.vp) + column;
        }
        // d_out's 64 rows of 32 columns: four elements a lane; lanes 0 .. 159 the factors of a product's column
        auto fetch = [&](int v0, int to) {
            const int tid = thread(), row = tid / 8, col = tid % 8 * 4;
            const Buffer outs = rows_at(o0, S.ot, steps, S.V);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t off = v0 + col + e < S.V ? (row * S.ot + v0 + col + e) * uint32_t(sizeof(E)) : NOWHERE;
                if constexpr (sizeof(E) == 2) op[e] = __builtin_amdgcn_raw_buffer_load_b16(outs.r, off, 0, 0);
                else op[e] = __builtin_amdgcn_raw_buffer_load_b32(outs.r, off, 0, 0);
            }
            if constexpr (HALF) {
                os = *reinterpret_cast<const f4*>(f1 + 2 * S.vp + v0 + col);
                lf = lp[v0];
                rf = rp[v0];
            }
            char* buffer = lds + IN + to * BUFFER;
            bring<WAVES>(b0 + v0 / COLS * Ke::BLOCK, buffer, BLOCK);
            bring<WAVES>(b1 + v0 / COLS * Ke::BLOCK, buffer + BLOCK, BLOCK);
        };
        auto put = [&](int to) {           // what went by way of registers
            const int tid = thread(), row = tid / 8, col = tid % 8 * 4;
            const Ot Od{reinterpret_cast<St*>(lds + IN + to * BUFFER + 2 * BLOCK)};
            pack<St, 4> x;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float d = Sixteen<E>::value(op[e]);
                x.v[e] = St(HALF ? d * __uint_as_float((254u << 23) - __float_as_uint(os[e])) : d);    // (over a power of two)
            }
            x.store(Od.p + row * Ot::ROW + place(col));
            if constexpr (HALF) if (tid < PRODUCTS * COLS) {
                const int e = exponent(lf) + exponent(rf) - most;      // 0 at most
                factors[to][tid / COLS][place(tid % COLS)] = e > -25 ? St(__uint_as_float((127 + e) << 23)) : St(0.0f);
            }
        };
        E gx, wx;                          // the gates of the lane's step
        {                                  // the steps' record, and the largest of the columns' scales by product: dO S, dR S, U dS, dO U, dR U
            const int tid = thread();
            const float* p = reinterpret_cast<const float*>(&reinterpret_cast<const Re*>(record_of<St>(const_cast<char*>(records), at))->steps);
            constexpr int N = int(sizeof(Steps) / 4), EACH = (N + MANY - 1) / MANY;
            float x[EACH];
#pragma unroll
            for (int k = 0; k < EACH; k++) x[k] = p[tid + k * MANY < N ? tid + k * MANY : N - 1];
            const int64_t t = t0 + (tid % WAVE < steps ? tid % WAVE : steps - 1);
            gx = gate[b * S.ab + t * S.at + g * S.ag];
            wx = write[b * S.wb + t * S.wt + g * S.wg];
            const int c0 = tid < S.vp ? tid : S.vp - 1;
            float scales[5];
            const auto read = [&](int c) {
                scales[0] = f0[c];
                scales[1] = f0[S.vp + c];
#pragma unroll
                for (int k = 0; k < 3; k++) scales[2 + k] = f1[k * S.vp + c];
            };
            if constexpr (HALF) read(c0);
            fetch(0, 0);
            fence();                       // (all of it is on its way)
            if constexpr (HALF) {
                int top[PRODUCTS];
#pragma unroll
                for (int p = 0; p < PRODUCTS; p++) top[p] = -1000;
                for (int c = c0;;) {
                    const int es = exponent(scales[0]), eu = exponent(scales[1]), ed = exponent(scales[2]), er = exponent(scales[3]), eo = exponent(scales[4]);
                    top[0] = max(top[0], eo + es);
                    top[1] = max(top[1], er + es);
                    top[2] = max(top[2], eu + ed);
                    top[3] = max(top[3], eo + eu);
                    top[4] = max(top[4], er + eu);
                    if ((c += MANY) >= S.vp) break;
                    read(c);
                }
#pragma unroll
                for (int p = 0; p < PRODUCTS; p++) {
                    top[p] = largest_of_wave(top[p]);
                    if (tid % WAVE == 0) tops[wave][p] = top[p];
                }
            }
#pragma unroll
            for (int k = 0; k < EACH; k++) if (tid + k * MANY < N) reinterpret_cast<float*>(&st)[tid + k * MANY] = x[k];
        }
        __syncthreads();
        if constexpr (HALF) {
            const int product = thread() / COLS < PRODUCTS ? thread() / COLS : 0;
            most = -1000;
#pragma unroll
            for (int w = 0; w < WAVES; w++) most = max(most, tops[w][product]);
        }
        put(0);
        if (j == 0) {                      // keys and queries come while the first block is used
            constexpr int BYTES = 2 * In::SIZE * int(sizeof(St));
            bring<WAVES>(images + (bh * S.chunks + chunk) * IN, lds, BYTES);
            arrived<(BYTES + 1024 * WAVES - 1) / (1024 * WAVES)>();
        } else {
            arrived<0>();
        }
        int now = 0;
        for (int v0 = 0; v0 < S.vp; v0 += COLS) {
            __syncthreads();               // the block is there, and the one before has been used
            const bool next = v0 + COLS < S.vp;
            const int tid = thread();
            St* buffer = reinterpret_cast<St*>(lds + IN + now * BUFFER);
            const Sv S0{buffer}, S1{buffer + Ke::BLOCK};
            const Uv Us{buffer + Sv::SIZE}, Rs{buffer + Ke::BLOCK + Sv::SIZE};
            const Ot Od{buffer + 2 * Ke::BLOCK};
            const auto scaled = [&](auto f, int p) {
                if constexpr (HALF) {
                    const h8 by = *reinterpret_cast<const h8*>(&factors[now][p][8 * (tid % WAVE / 16)]);
#pragma unroll
                    for (auto& part : f.p) part *= by;
                }
                return f;
            };
            if (BUFFERS == 2 && next) fetch(v0 + COLS, now ^ 1);
            // operands of two parts are loaded in two stages, where all at once have no room
            const auto of = Od.rows(band, 0);
            const auto rf = Rs.cols(band, 0);
            Frag<St, WIDE> sf[ND], gf[ND], un[2];
#pragma unroll
            for (int n = 0; n < ND; n++) sf[n] = S0.cols(d0 + 16 * n, 0);
#pragma unroll
            for (int k = 0; k < 2; k++) un[k] = Us.cols(16 * (half + 2 * k), 0);
            float product[2] = {0.0f, 0.0f};
            constexpr int UNITS = COLS * DK / UNIT, EACH = (UNITS + MANY - 1) / MANY;
#pragma unroll
            for (int k = 0; k < EACH; k++) {
                const int p = tid + k * MANY < UNITS ? tid + k * MANY : 0, c = p / (DK / UNIT), at = c * Sv::ROW + p % (DK / UNIT) * UNIT;
                float z = 0.0f;
#pragma unroll
                for (int i = WIDE - 1; i >= 0; i--)
#pragma unroll
                    for (int j = WIDE - 1; j >= 0; j--) if (i + j < WIDE) {
                        const auto x = pack<St, UNIT>::load(S0.p + i * Sv::PLANE + at), y = pack<St, UNIT>::load(S1.p + j * Sv::PLANE + at);
#pragma unroll
                        for (int e = 0; e < UNIT; e++) if constexpr (!HALF) z = fmaf(x.v[e], y.v[e], z);
                        if constexpr (HALF) {
                            using h2 = __attribute__((ext_vector_type(2))) _Float16;
#pragma unroll
                            for (int e = 0; e < UNIT; e += 2) z = __builtin_amdgcn_fdot2(h2{x.v[e], x.v[e + 1]}, h2{y.v[e], y.v[e + 1]}, z, false);
                        }
                    }
                if constexpr (HALF) z = ldexpf(z, exponent(f0[v0 + c]) + exponent(f1[v0 + c]));        // (their product may be past float32 where z is 0)
                product[k % 2] += tid + k * MANY < UNITS ? z : 0.0f;
            }
            both += product[0] + product[1];
            fence();
            const auto of0 = scaled(of, 0), of3 = scaled(of, 3);
            const auto rf1 = scaled(rf, 1), rf4 = scaled(rf, 4);
#pragma unroll
            for (int k = 0; k < 2; k++) {  // (those above the diagonal are not used)
                mma(dp[k], of3, un[k]);
                mma(da[k], rf4, un[k]);
            }
            const auto uf = Us.cols(band, 0);
#pragma unroll
            for (int n = 0; n < ND; n++) gf[n] = S1.cols(d0 + 16 * n, 0);
#pragma unroll
            for (int n = 0; n < ND; n++) {
                mma(aq[n], of0, sf[n]);
                mma(from[n], rf1, sf[n]);
            }
            fence();
            const auto uf2 = scaled(uf, 2);
#pragma unroll
            for (int n = 0; n < ND; n++) mma(to[n], uf2, gf[n]);
            if (next) {
                if constexpr (BUFFERS == 1) {
                    __syncthreads();
                    fetch(v0 + COLS, 0);
                }
                put(BUFFERS == 2 ? now ^ 1 : 0);
                arrived<0>();
                if (BUFFERS == 2) now ^= 1;
            }
        }
        if (j == 0) {
            arrived<0>();                  // keys and queries, of all waves
            __syncthreads();
        }
        int top[PRODUCTS];
#pragma unroll
        for (int p = 0; p < PRODUCTS; p++) {
            top[p] = HALF ? -1000 : 0;
            if constexpr (HALF) {
#pragma unroll
                for (int w = 0; w < WAVES; w++) top[p] = max(top[p], tops[w][p]);
            }
        }
        const uint64_t cuts = uint64_t(st.cut[1]) << 32 | st.cut[0];
        const int tid = thread(), l = tid % WAVE, grp = l / 16, m = l % 16;
        // what a step has of the state before the chunk and leaves after it, and its row's sums
        const f4 hi = *reinterpret_cast<const f4*>(st.hi + band + 4 * grp), lo = *reinterpret_cast<const f4*>(st.lo + band + 4 * grp);
        const f4 bi = *reinterpret_cast<const f4*>(st.b + band + 4 * grp);
        f4 rki = *reinterpret_cast<const f4*>(st.rk + band + 4 * grp), rqi = *reinterpret_cast<const f4*>(st.rq + band + 4 * grp), rowsum;
        const float last_hi = st.hi[C - 1], last_lo = st.lo[C - 1];
        const int last_cut = since(cuts, C - 1);
        int since_i[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = band + 4 * grp + r;
            since_i[r] = since(cuts, i);
            const float gi = since_i[r] >= 0 ? 0.0f : decay<St>(hi[r]), li = i < last_cut ? 0.0f : decay<St>((last_hi - hi[r]) + (last_lo - lo[r]));
            rki[r] = length_rest<St>(rki[r]);
            rqi[r] = length_rest<St>(rqi[r]);
            float q[ND], k[ND], dq = 0.0f, df = 0.0f, dt = 0.0f;
#pragma unroll
            for (int n = 0; n < ND; n++) {
                q[n] = float(Qt.get(i, d0 + 16 * n + m));
                k[n] = float(Kt.get(i, d0 + 16 * n + m));
            }
#pragma unroll
            for (int n = 0; n < ND; n++) {
                const float x = part_of_it<true>(gi, ldexpf(aq[n][r], top[0])), y = part_of_it<true>(-bi[r] * gi, ldexpf(from[n][r], top[1]));
                const float z = part_of_it<true>(li, ldexpf(to[n][r], top[2]));
                dq = fmaf(q[n], x, dq);
                df = fmaf(k[n], y, df);
                dt = fmaf(k[n], z, dt);
                tq[n][r] += x;
                tk[n][r] += y + z;
            }
            rowsum[r] = rqi[r] * dq + rki[r] * df;
            dt = over_row(dt);
            if (m == 0) left[half][i] = rki[r] * dt;
        }
        f4 kk[2] = {zero, zero}, qk[2] = {zero, zero};
#pragma unroll
        for (int kb = 0; kb < KB; kb++) {
            const auto ka = Kt.rows(band, kb), qa = Qt.rows(band, kb);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const auto kn = Kt.rows(16 * (half + 2 * k), kb);
                mma(kk[k], ka, kn);
                mma(qk[k], qa, kn);
            }
        }
        both = over_row(sum_over_rows(both));
        if (l == 0) whole[wave] = both;
        __syncthreads();                   // the last block of values has been used
        // E and F with the lengths of what they are multiplied by, F on both sides of the diagonal
        // (dp and da are 2^28 V at most, a length's rest 2 / LONG: what is left is 2^14)
        constexpr float FIT = HALF ? 0x1p-15f * LONG<St> : 1.0f;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int n = half + 2 * k, c = 16 * n + m, at = place(c);
            float column = 0.0f;
            if (n > own) {                 // above the diagonal
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    put_parts(Ek, band + 4 * grp + r, at, 0.0f);
                    put_parts(Eq, band + 4 * grp + r, at, 0.0f);
                }
            } else {
                const float rk = length_rest<St>(st.rk[c]), hc = st.hi[c], lc = st.lo[c];
                f4 fk;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = band + 4 * grp + r;
                    const bool on = c <= i && c >= since_i[r];
                    const float M = decay<St>(on ? (hi[r] - hc) + (lo[r] - lc) : 0.0f);
                    const float e = on ? M * dp[k][r] : 0.0f, f = on && c < i ? -M * bi[r] * da[k][r] : 0.0f;
                    const float pair = c < i ? ldexpf(e * rqi[r] * rk * qk[k][r], top[3]) + ldexpf(f * rki[r] * rk * kk[k][r], top[4]) : 0.0f;
                    rowsum[r] += pair;
                    column += pair;
                    put_parts(Ek, i, at, e * (few * FIT) * rk);
                    put_parts(Eq, i, at, e * (few * FIT) * rqi[r]);
                    if (n < own || c <= i) put_parts(Ff, i, at, f * (few * FIT) * rk);
                    fk[r] = f * (few * FIT) * rki[r];
                }
                if (n < own) {             // the four steps' places are neighbours
                    pack<St, 4> x;
#pragma unroll
                    for (int w = 0; w < WIDE; w++) {
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            x.v[r] = St(fk[r]);
                            fk[r] -= float(x.v[r]);
                        }
                        x.store(Ff.p + w * Square::PLANE + c * Square::ROW + place(band + 4 * grp));
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int i = band + 4 * grp + r;
                        if (c < i) put_parts(Ff, c, place(i), fk[r]);
                        if (c == i) writes[i] = ldexpf(da[k][r], top[4]);
                    }
                }
                column = sum_over_rows(column);
            }
            if (grp == 0) columns[own][c] = column;
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float x = over_row(rowsum[r]);
            if (m == 0) rows[half][band + 4 * grp + r] = x;
        }
        __syncthreads();
        constexpr int OUT = HALF ? 15 - 6 : 0;             // (what FIT took out)
        static_assert(!HALF || LONG<St> == 64.0f, "the exponent of LONG");
        Frag<St, WIDE> ek[2], eq[2], ff[2];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            ek[kb] = Ek.rows(band, kb);
            eq[kb] = Eq.cols(band, kb);
            ff[kb] = Ff.rows(band, kb);
        }
#pragma unroll
        for (int n = 0; n < ND; n++) {
            f4 x = zero, y = zero, z = zero;
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                const auto kn = Kt.cols(d0 + 16 * n, kb);
                mma(x, ek[kb], kn);
                mma(z, ff[kb], kn);
                mma(y, eq[kb], Qt.cols(d0 + 16 * n, kb));
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                tq[n][r] += ldexpf(x[r], top[3] + many + OUT);
                tk[n][r] += ldexpf(y[r], top[3] + many + OUT) + ldexpf(z[r], top[4] + many + OUT);
            }
        }
        // a lane for each step: what its gate gets from the pairs around it and from the states, by two waves
        if (wave == 0) {
            const auto same = [&](int i) { return i < C && since(cuts, i) <= l; };     // no step up to i, from the next on, drops the state
            double after = double(rows[0][l]) + rows[1][l] - (double(columns[0][l]) + columns[1][l] + columns[2][l] + columns[3][l]);
#pragma unroll
            for (int d = 1; d < WAVE; d <<= 1) {
                const double x = __shfl_down(after, d, WAVE);
                if (same(l + d)) after += x;
            }
            gates[0][l] = after;
        } else if (wave == 1) {
            double before = double(left[0][l]) + left[1][l];
#pragma unroll
            for (int d = 1; d < WAVE; d <<= 1) {
                const double x = __shfl_up(before, d, WAVE);
                if (l >= d) before += x;
            }
            before = __shfl_up(before, 1, WAVE);
            if (l == 0) before = 0.0;
            if (since(cuts, l) < 0 && st.end != 0.0f) {
                double sum = 0.0;
#pragma unroll
                for (int w = 0; w < WAVES; w++) sum += whole[w];
                before += double(st.end) * sum;
            }
            gates[1][l] = before;
        }
        __syncthreads();
        if (wave == 0 && l < steps) {
            const int64_t to = (b * S.T + t0 + l) * S.G + g;
            d_gate[to] = E(cuts >> l & 1 ? 0.0f : -float(gates[0][l] + gates[1][l]) / (1.0f + expf(-float(gx))));
            d_write[to] = E(writes[l] / (1.0f + expf(float(wx))));
        }
    }
    // of the query and the key themselves: d - x^ (x^.d), over the length
    const int l = thread() % WAVE, grp = l / 16, m = l % 16;
    f4 rk = *reinterpret_cast<const f4*>(st.rk + band + 4 * grp), rq = *reinterpret_cast<const f4*>(st.rq + band + 4 * grp);
    const uint64_t odd = uint64_t(st.odd[1]) << 32 | st.odd[0], queries = uint64_t(st.odd_query[1]) << 32 | st.odd_query[0];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int i = band + 4 * grp + r;
        if ((odd | queries) >> i & 1) rk[r] = NAN;     // (a query that is not finite reaches its own step's key by way of the state)
        if (queries >> i & 1) rq[r] = NAN;
        float dq = 0.0f, dk = 0.0f;
#pragma unroll
        for (int n = 0; n < ND; n++) {
            dq = fmaf(float(Qt.get(i, d0 + 16 * n + m)), tq[n][r], dq);
            dk = fmaf(float(Kt.get(i, d0 + 16 * n + m)), tk[n][r], dk);
        }
        dq = over_row(dq);
        dk = over_row(dk);
        if (m == 0) {
            dots[0][half][i] = dq;
            dots[1][half][i] = dk;
        }
    }
    __syncthreads();
    const Buffer dq0 = rows_at(d_query + ((b * S.T + t0) * S.H + h) * S.K, S.H * S.K, steps, S.K), dk0 = rows_at(d_key + ((b * S.T + t0) * S.H + h) * S.K, S.H * S.K, steps, S.K);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int i = band + 4 * grp + r;
        const float rkr = length_rest<St>(rk[r]), rqr = length_rest<St>(rq[r]);
        const float dq = (dots[0][0][i] + dots[0][1][i]) * rqr * rqr, dk = (dots[1][0][i] + dots[1][1][i]) * rkr * rkr;
#pragma unroll
        for (int n = 0; n < ND; n++) {
            const int c = d0 + 16 * n + m;
            const uint32_t to = c < S.K ? (i * S.H * S.K + c) * uint32_t(sizeof(E)) : NOWHERE;
            dq0.store(E(rq[r] * fmaf(-dq, float(Qt.get(i, c)), tq[n][r])), to);
            dk0.store(E(rk[r] * fmaf(-dk, float(Kt.get(i, c)), tk[n][r])), to);
        }
    }
}

// The same backwards. A workgroup of four waves and the one that brings has two on a SIMD, which are held to 256 registers each; with keys of
// over 64 elements a wave backwards takes more, and spills cost more than two waves do. All of a backward pass, ms, with two and with four: 128 heads of 128 x 128,
// 8,192 steps, bfloat16 2.85 and 2.93, float32 6.25 and 7.53; 192 heads 4.25 and 4.84; 256 heads of 64 x 64, 4,096 steps, bfloat16 1.51 and 1.48, float32 2.40
// and 1.99.
template <int DK, typename F> int32_t with_waves_back(const Shape& S, const Pieces& pieces, F&& f) {
    if constexpr (DK > 64) return f(std::integral_constant<int, 2>{});
    else return with_waves(S, pieces, f);
}
// And for the walk of pieces from zero, which has no columns beside those of values: two where the workgroups are no more than CUs. One
// sequence of 32,768 steps, ms, with two and with four: 4 heads of 128 x 128 bfloat16 0.55 and 0.59, float32 1.22 and 1.59; past the CUs, 2 heads of 128 x 512
// bfloat16 1.00 and 0.92, 8 heads of 64 x 128 float32 2.12 and 1.75.
template <typename F> int32_t with_waves_from_zero(const Shape& S, const Pieces& pieces, F&& f) {
    if (pieces.count * S.B * S.G * (S.vp / 32) <= 256) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 4>{});
}

template <typename E, int DK>
int32_t backward(const void* gate, const void* write, const void* d_out, const float* d_last, const Shape& S, void* kept, const void* records, void* d_query, void* d_key,
                 void* d_value, void* d_gate, void* d_write, float* d_state, void* work, hipStream_t stream, char* err, size_t errcap) {
    using St = Rep<E>;
    const auto in = [](const void* p) { return static_cast<const E*>(p); };
    const auto out = [](void* p) { return static_cast<E*>(p); };
    const int64_t heads = S.B * S.G;
    const char *rec = static_cast<const char*>(records), *images = rec + heads * S.chunks * Record<St>::STRIDE;
    const Kept<St, DK> before(kept, S), walked(work, S);
    const Pieces pieces = pieces_of(heads, S.chunks, S.vp, DK);
    const Joins maps(const_cast<char*>(images) + S.B * S.H * S.chunks * IMAGE<St, DK>, heads, pieces.count, S.vp, DK);
    const Joins joins(walked.scales + heads * S.chunks * 3 * S.vp, heads, pieces.count, S.vp, DK);
    if (pieces.count > 1) {
        with_waves_from_zero(S, pieces, [&](auto w) {
            constexpr int W = decltype(w)::value;
            walk_kernel<E, DK, W, true><<<dim3(heads * pieces.count * ((S.vp / 16 + W - 1) / W)), (W + 1) * WAVE, 0, stream>>>(in(d_out), nullptr, S, rec, images, nullptr,
                                                                                                                          nullptr, walked, pieces, joins);
            return 0;
        });
        join_kernel<DK, true><<<dim3(heads * (S.vp / 16)), (JOIN_WAVES + 1) * WAVE, 0, stream>>>(d_last, S, pieces.count, joins, maps);
    }
    with_waves_back<DK>(S, pieces, [&](auto w) {
        constexpr int W = decltype(w)::value;
        walk_kernel<E, DK, W, false><<<dim3(heads * pieces.count * ((S.vp / 16 + W - 1) / W)), (W + 1) * WAVE, 0, stream>>>(in(d_out), d_last, S, rec, images, out(d_value),
                                                                                                                       d_state, walked, pieces, joins);
        return 0;
    });
    gradient_kernel<E, DK><<<dim3(S.B * S.H * S.chunks), MANY, 0, stream>>>(in(gate), in(write), in(d_out), S, rec, images, before, walked, out(d_query), out(d_key),
                                                                           out(d_gate), out(d_write));
    return launched(err, errcap);
}

}  // namespace

extern "C" int32_t pv_gated_delta_backward_hip(const void* gate, const void* write, const void* d_out, const float* d_last, int64_t B, int64_t T, int32_t H, int32_t G,
                                               int32_t K, int32_t V, const int64_t* strides, int32_t dtype, const void* kept, const void* records, void* d_query,
                                               void* d_key, void* d_value, void* d_gate, void* d_write, float* d_state, void* work, uint64_t work_bytes, void* stream,
                                               char* err, size_t errcap) {
    Shape S;
    if (int32_t e = shape_of(B, T, H, G, K, V, strides, 9, 0.0f, dtype, S, err, errcap)) return e;
    if (!gate || !write || !d_out || !kept || !records || !d_query || !d_key || !d_value || !d_gate || !d_write) return fail(PV_EARG, err, errcap, "null argument");
    if (!aligned(kept, 16) || !aligned(records, 16)) return fail(PV_EARG, err, errcap, "kept, records: not 16-byte aligned");
    const uint64_t need = pv_gated_delta_backward_work_bytes(B, T, G, K, V, dtype);
    if (!work || work_bytes < need || !aligned(work, 16)) return fail(PV_EARG, err, errcap, "work: too small, or not 16-byte aligned");
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        return with_k(K, [&](auto k) {
            return backward<E, decltype(k)::value>(gate, write, d_out, d_last, S, const_cast<void*>(kept), records, d_query, d_key, d_value, d_gate, d_write, d_state, work,
                                                   hipStream_t(stream), err, errcap);
        });
    });
}
