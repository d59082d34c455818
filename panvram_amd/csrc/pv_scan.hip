// Gated linear recurrence h[t] = (1 - z[t]) h[t-1] + z[t] value[t], z = sigmoid(gate), over [B, T, D], and its gradients.
//
// A run of steps is the map h -> A h + H of the state before it: A the product of its (1 - z), H the run started at zero.
// Maps of neighbouring runs join, so all of T is worked on at once and every byte is read once and written once:
//   - a wave holds STEPS steps of 64 x VEC channels in registers, a workgroup of WAVES waves a chunk of WAVES x STEPS steps;
//   - the workgroup makes its chunk's map, publishes it (`Before`), joins the maps of the chunks before, and walks its
//     steps from there.
// The gradient is the same recurrence backwards: C[t] = (1 - z[t]) (d_out[t] + C[t+1]), C what flows into h[t-1]; the states
// before each step are made again from the start of the wave's steps, which the forward pass leaves in `carry` (one f32 for
// SPAN steps of a channel, so that h is never read). A step's arithmetic is the same for every cut of T, and so is the order in which maps are
// joined: results do not depend on which workgroup was faster.
//
// A reset at t drops h[t-1], whatever it holds (a NaN too): the step is chosen, not multiplied by zero, and the map of a run
// with a reset in it has A = CUT, which no product of (1 - z) can be.
//
// What bounds it: the bytes, three tensors forwards and five backwards. In bfloat16 the arithmetic is next (two transcendental
// and some 25 other operations an element forwards, 40 backwards, at 16 waves a CU), and in long sequences the wait for
// the maps of chunks that are still being loaded. Measured: 8 x 8,192 x 1,024 bfloat16 forwards 88-91 us (403 MB: 4.4-4.6 TB/s),
// backwards 128-133 us (671 MB: 5.0-5.2); in float32 152 and 250 (5.3 and 5.4 TB/s); 1 x 2^20 x 512 bfloat16 forwards 618-631 us
// (5.1 TB/s); one step of 16 x 1,024 3.3 us, a launch.
#include "pv_ops.h"

using namespace pvo;

namespace {

// Steps of a wave, whose loads are all in flight at once, and waves of a workgroup where T has more steps than a wave. Forwards 32
// (1 x 2^20 x 512 bfloat16 in 640 us; 745 with 16, whose maps are twice as many), 4 for sequences that short (a single step is
// all launch); backwards, with one tensor more to hold, 16.
constexpr int STEPS_FORWARD = 32, STEPS_BACK = 16, STEPS_SHORT = 4, CHUNK_WAVES = 8;
constexpr int SPAN = 16;                   // steps from one state that is kept for the backward pass to the next
static_assert(SPAN == STEPS_BACK && STEPS_FORWARD % SPAN == 0, "a wave of the backward pass starts at a state that is kept");
constexpr float CUT = -1.0f;

struct Shape {
    int64_t B, T, D, gb, gt, vb, vt, db, dt;   // strides in elements: gate, value, d_out (batch, time); channels are neighbours
    int64_t ot;                                // of the outputs' steps: D
    int64_t spans, chunks, tiles;              // spans of SPAN and chunks of T, tiles of D
};

// z = sigmoid(g) and k = 1 - z of a step in one register: the smaller of the two, its sign bit set where that is z. It is made from
// exp(-|g|); the other is 1 minus it, at least a half and so as exact. -0: z = 0, k = 1.
// Gates in 32 bits: exp(-a) = 2^t (1 + ln2 r), t = a log2(e) rounded and r what the rounding left, good to a few units in the last
// place. Gates in 16 bits: 2^t alone, off by some |g| 2^-24 of itself, where the gate's own rounding to 16 bits has moved z by some
// |g| 2^-12 or more. (The correction costs 8 x 8,192 x 1,024 nothing in float32, 152 us either way, and in bfloat16 96 us for 93.)
template <typename E> __device__ inline float gate_of(float g) {
    float e;
    if constexpr (sizeof(E) == 4) {
        constexpr float L = 1.44269504f, REST = 1.9259630e-8f, LN2 = 0.69314718f;      // log2(e) = L + REST
        float a = fabsf(g);
        a = a > 127.0f ? 127.0f : a;       // (exp(-127) is 0 here; a NaN stays)
        const float t = -L * a, p = __builtin_amdgcn_exp2f(t);
        e = fmaf(p, LN2 * fmaf(-REST, a, fmaf(-L, a, -t)), p);
    } else {
        e = __expf(-fabsf(g));
    }
    return copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), g);
}
__device__ inline void both(float q, float& z, float& k) {
    const float a = fabsf(q), b = 1.0f - a;
    const bool low = int32_t(__float_as_uint(q)) < 0;
    z = low ? a : b;
    k = low ? b : a;
}

struct Map { float A, H; };
__device__ inline float apply(Map m, float before) { return m.A == CUT ? m.H : fmaf(m.A, before, m.H); }
__device__ inline Map then(Map first, Map second) {
    return {first.A == CUT || second.A == CUT ? CUT : first.A * second.A, apply(second, first.H)};
}

// A wave has 64 x VEC channels from d0 on, slot VEC * lane + v. The last lane of an odd D takes channel D - 2 once more beside the
// last one: it computes and writes what its neighbour does.
template <int VEC> __device__ inline int64_t channel_of(int64_t D, int64_t d0, int slot) {
    int64_t d = d0 + slot / VEC * VEC;
    if (VEC > 1 && d + VEC > D) d = D - VEC;
    return d + slot % VEC;
}
template <int VEC> __device__ inline bool is_channel(int64_t D, int64_t d0, int slot) { return d0 + slot / VEC * VEC < D; }

// ---- Maps of chunks, in the order of the walk (position 0 first), passed between workgroups.
// Level 0 has a map for each chunk, level l + 1 one for each FAN whole neighbours of level l. The workgroup at position p needs
// the maps of its predecessors within its group of FAN, of their group's predecessors within its, and so on: the base-FAN
// digits of p, at most FAN - 1 maps a level. The last of a group makes the group's map of them and its own.
//
// A map is one 8-byte word (A, H) per channel, written by one store; EMPTY until then. Its NaNs are stored as 0x7fc00000, so
// that no map is EMPTY. A word is read and written past the L2 caches (agent scope); no other data depends on the order.
// Every wait ends: a workgroup takes its position from a counter, so all earlier positions belong to workgroups that run
// already, a position publishes level 0 without waiting, and each other level after waiting for earlier positions only. (Should a word not come in some seconds all the same, it counts as NaN.)
constexpr int FAN = 8, LEVELS = 8;         // 8^8 chunks
constexpr uint64_t EMPTY = ~0ull;
constexpr int POLLS = 1 << 22;

struct Records {
    uint32_t* next;                        // the position and tile to hand out next
    uint64_t* level[LEVELS];
};

__global__ __launch_bounds__(256) void records_kernel(uint64_t* words, int64_t n) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) words[i] = i < 2 ? 0 : EMPTY;
}

__device__ inline uint64_t word_of(float A, float H) {
    const uint32_t a = A != A ? 0x7fc00000u : __float_as_uint(A), h = H != H ? 0x7fc00000u : __float_as_uint(H);
    return uint64_t(h) << 32 | a;
}
__device__ inline void publish(uint64_t* at, Map m, bool on) {
    if (on) __hip_atomic_store(at, word_of(m.A, m.H), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The maps of a group's first members on level l, up to position p of that level, joined in order; for the lane's channel d (on)
__device__ inline Map before_at(const Records& R, const Shape& S, int64_t b, int l, int64_t n, int64_t p, int64_t d, bool on) {
    const int many = int(p & (FAN - 1));
    const uint64_t* rec = R.level[l] + (b * n + (p - many)) * S.D + d;
    uint64_t w[FAN - 1];
#pragma unroll
    for (int i = 0; i < FAN - 1; i++) {
        w[i] = 0;
        if (i < many && on) w[i] = __hip_atomic_load(rec + i * S.D, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    Map all = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < FAN - 1; i++) {
        if (i >= many) break;
        for (int k = 0; __any(w[i] == EMPTY) && k < POLLS; k++) {
            __builtin_amdgcn_s_sleep(1);
            if (on) w[i] = __hip_atomic_load(rec + i * S.D, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        all = then(all, {__uint_as_float(uint32_t(w[i])), __uint_as_float(uint32_t(w[i] >> 32))});
    }
    return all;
}

// ---- What a workgroup works on: channels d.. of sequence b, position p of the walk
template <int VEC, int WAVES, bool ONE> struct Place {
    int64_t b, p, d0, d;                   // d: the lane's first channel, d0: the wave's
    int wave, lane;
    bool on;
    __device__ Place(const Shape& S, const Records& R) {
        lane = threadIdx.x % WAVE;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
        uint32_t turn = blockIdx.x;
        if constexpr (!ONE) {
            __shared__ uint32_t given;
            if (threadIdx.x == 0) given = __hip_atomic_fetch_add(R.next, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            turn = __builtin_amdgcn_readfirstlane(given);
        }
        const uint32_t rows = uint32_t(S.B * S.tiles);
        const uint32_t q = __builtin_amdgcn_readfirstlane(turn / rows), rest = turn - q * rows;
        const uint32_t c = __builtin_amdgcn_readfirstlane(rest / uint32_t(S.tiles));
        p = q;
        b = c;
        d0 = int64_t(rest - c * uint32_t(S.tiles)) * (WAVE * VEC);
        if (S.D - d0 < VEC) d0 = S.D - VEC;    // (one channel left over: with its neighbour)
        d = channel_of<VEC>(S.D, d0, lane * VEC);
        on = is_channel<VEC>(S.D, d0, lane * VEC);
    }
};

// A wave's steps [t0, t0 + steps), and a bit for each that has a reset
struct Span { int64_t t0; int steps; uint32_t cuts; };
template <int STEPS> __device__ inline Span span_of(const Shape& S, const uint8_t* reset, int64_t b, int64_t t0, int lane) {
    Span s;
    s.t0 = t0;
    const int64_t left = S.T - t0;
    s.steps = left <= 0 ? 0 : left < STEPS ? int(left) : STEPS;
    s.cuts = 0;
    if (reset) s.cuts = uint32_t(__ballot(lane < s.steps && reset[b * S.T + t0 + lane] != 0));
    return s;
}
// (from is the same for the wave, at: the lane's channel in it)
// A wave's steps of a tensor as a buffer of its rows: step i is at i * stride bytes, and what lies behind the span (or at NO_LANE)
// is not read and not written, so that neither the end of T nor that of D needs a branch. Rows may begin at any element: gfx950
// takes a 4-byte access at 2 bytes' alignment.
constexpr uint32_t NO_LANE = 1u << 31;
// ONCE: accesses with the hint that the data is not used again soon (`once_of` says when)
constexpr int64_t MOST_STRIDE = 1 << 26;   // bytes: the offsets of a wave's steps stay below 2^31
template <bool ONCE> struct Rows {
    static constexpr int HINT = ONCE ? 2 : 0;
    __amdgpu_buffer_rsrc_t buffer;
    int stride;
    template <typename E> __device__ Rows(const E* from, int64_t step, const Span& s, int64_t channels) {
        stride = int(step * int64_t(sizeof(E)));
        const int bytes = s.steps ? (s.steps - 1) * stride + int(channels * int64_t(sizeof(E))) : 0;
        buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(from + s.t0 * step), 0, bytes, 0x00027000);
    }
    template <int BYTES> __device__ uint32_t load(int i, uint32_t at) const {
        if constexpr (BYTES == 4) return __builtin_amdgcn_raw_buffer_load_b32(buffer, at, i * stride, HINT);
        else return __builtin_amdgcn_raw_buffer_load_b16(buffer, at, i * stride, HINT);
    }
    template <int BYTES> __device__ void store(uint32_t bits, int i, uint32_t at) const {
        if constexpr (BYTES == 4) __builtin_amdgcn_raw_buffer_store_b32(bits, buffer, at, i * stride, HINT);
        else __builtin_amdgcn_raw_buffer_store_b16(uint16_t(bits), buffer, at, i * stride, HINT);
    }
};

// A step's VEC values in one register, as they lie in memory. (As elements the compiler would give each a register.)
template <typename E, int VEC> struct Word {
    static constexpr int BYTES = VEC * int(sizeof(E));
    static_assert(BYTES <= 4, "one register");
    uint32_t bits;
    __device__ float get(int v) const {
        if constexpr (sizeof(E) == 4) return __uint_as_float(bits);
        else if constexpr (std::is_same_v<E, bf16>) return __uint_as_float(v ? bits & 0xffff0000u : bits << 16);
        else return float(__builtin_bit_cast(f16, uint16_t(bits >> 16 * v)));
    }
    static __device__ Word of(const float* x) {
        if constexpr (sizeof(E) == 4) return {__float_as_uint(x[0])};
        else if constexpr (VEC == 1) return {__builtin_bit_cast(uint16_t, E(x[0]))};
        else {
            using F2 = __attribute__((ext_vector_type(2))) float;
            using E2 = __attribute__((ext_vector_type(2))) E;
            return {__builtin_bit_cast(uint32_t, __builtin_convertvector((F2{x[0], x[1]}), E2))};
        }
    }
};
template <int STEPS, typename E, int VEC, bool ONCE> __device__ inline void load_steps(Word<E, VEC> (&to)[STEPS], const Rows<ONCE>& rows, uint32_t at) {
#pragma unroll
    for (int i = 0; i < STEPS; i++) to[i].bits = rows.template load<Word<E, VEC>::BYTES>(i, at);
}
// Behind the end: gates that leave the state as it is (z = 0), zeros in the other tensors. (A buffer's zeros are no such thing
// for the gates, and are not there where all steps are one and the same row, stride 0.)
template <int STEPS, typename E, int VEC> __device__ inline void end_steps(Word<E, VEC> (&x)[STEPS], const Span& s, float rest) {
    if (s.steps == STEPS) return;
    const float both[2] = {rest, rest};
#pragma unroll
    for (int i = 0; i < STEPS; i++) if (i >= s.steps) x[i] = Word<E, VEC>::of(both);
}
// The compiler is to make what follows from these registers again where it needs it: kept from one walk over the steps to the
// next, z, 1 - z and the products would take two to four times the registers
template <int STEPS, int VEC> __device__ inline void anew(float (&q)[STEPS][VEC]) {
#pragma unroll
    for (int i = 0; i < STEPS; i++)
#pragma unroll
        for (int v = 0; v < VEC; v++) asm volatile("" : "+v"(q[i][v]));
}
template <int STEPS, typename E, int VEC> __device__ inline void anew(Word<E, VEC> (&x)[STEPS]) {
#pragma unroll
    for (int i = 0; i < STEPS; i++) asm volatile("" : "+v"(x[i].bits));
}
// f(i, whether step i has a reset) over the steps in order or backwards
template <int STEPS, bool RESET, bool BACK, typename F> __device__ inline void over_steps(const Span& s, F&& f) {
#pragma unroll
    for (int i = 0; i < STEPS; i++) { const int k = BACK ? STEPS - 1 - i : i; f(k, RESET && (s.cuts >> k & 1)); }
}

// The maps of the chunks before a workgroup's, level by level and by channel. VEC waves, of 64 channels each, have a level: all
// levels are waited for at once.
template <int VEC, int WAVES> struct Before {
    int levels;                            // of the chunks
    pack<float, VEC> A[LEVELS][WAVE], H[LEVELS][WAVE];

    // own: the chunk's map, wanted of the first VEC waves. Those have level 0, and where they are the last of a group they make the
    // group's map of its members' and their own at once, and so on up: no map waits for one of a higher level.
    __device__ void wait(const Records& R, const Shape& S, int64_t b, int64_t p, int64_t d0, int wave, int lane, Map own) {
        constexpr int TEAMS = WAVES / VEC;
        const int c = wave % VEC * WAVE + lane, team = wave / VEC;
        const int64_t d = channel_of<VEC>(S.D, d0, c);
        const bool on = is_channel<VEC>(S.D, d0, c);
        if (team == 0) publish(R.level[0] + (b * S.chunks + p) * S.D + d, own, on);
        int64_t n = S.chunks;
        int l = 0;
        for (bool whole = team == 0; l < LEVELS && n > 0; l++, n /= FAN, p /= FAN) {
            if (!whole && l % TEAMS != team) continue;
            const Map m = before_at(R, S, b, l, n, p, d, on);
            if (l % TEAMS == team) {
                A[l][c / VEC].v[c % VEC] = m.A;
                H[l][c / VEC].v[c % VEC] = m.H;
            }
            whole = whole && p % FAN == FAN - 1 && l + 1 < LEVELS;
            if (whole) {
                own = then(m, own);
                publish(R.level[l + 1] + (b * (n / FAN) + p / FAN) * S.D + d, own, on);
            }
        }
        levels = l;
    }
    __device__ float from(float first, int lane, int v) const {
        for (int l = levels - 1; l >= 0; l--) first = apply({A[l][lane].v[v], H[l][lane].v[v]}, first);
        return first;
    }
};

// The waves' maps of a chunk, by channel
template <int VEC, int WAVES> struct Maps {
    pack<float, VEC> A[WAVES][WAVE], H[WAVES][WAVE];
    __device__ void put(int wave, int lane, const Map* m) {
#pragma unroll
        for (int v = 0; v < VEC; v++) { A[wave][lane].v[v] = m[v].A; H[wave][lane].v[v] = m[v].H; }
    }
    __device__ Map get(int wave, int channel) const { return {A[wave][channel / VEC].v[channel % VEC], H[wave][channel / VEC].v[channel % VEC]}; }
};

template <typename E, int VEC, int STEPS, int WAVES, bool ONE, bool RESET, bool ONCE>
__global__ __launch_bounds__(WAVES* WAVE) __attribute__((amdgpu_waves_per_eu(VEC == 2 && WAVES > 1 ? 4 : 1))) void scan_kernel(Shape S, Records R, const E* __restrict__ gate, const E* __restrict__ value,
                                                           const float* __restrict__ state, const uint8_t* __restrict__ reset, E* __restrict__ out,
                                                           float* __restrict__ last, float* __restrict__ carry) {
    __shared__ Maps<VEC, WAVES> maps;
    __shared__ Before<VEC, WAVES> before;
    const Place<VEC, WAVES, ONE> P(S, R);
    const Span s = span_of<STEPS>(S, reset, P.b, (P.p * WAVES + P.wave) * STEPS, P.lane);
    const uint32_t at = P.on ? uint32_t(P.d - P.d0) * sizeof(E) : NO_LANE;
    const int64_t width = S.D - P.d0 < WAVE * VEC ? S.D - P.d0 : WAVE * VEC;
    Word<E, VEC> g[STEPS], x[STEPS];
    load_steps(g, Rows<ONCE>(gate + P.b * S.gb + P.d0, S.gt, s, width), at);
    load_steps(x, Rows<ONCE>(value + P.b * S.vb + P.d0, S.vt, s, width), at);
    end_steps(g, s, -INFINITY);
    end_steps(x, s, 0.0f);
    float Z[STEPS][VEC], h[VEC];
    if constexpr (WAVES > 1) {
        Map m[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) m[v] = {1.0f, 0.0f};
        over_steps<STEPS, RESET, false>(s, [&](int i, bool cut) {
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                Z[i][v] = gate_of<E>(g[i].get(v));
                float z, k;
                both(Z[i][v], z, k);
                const float in = z * x[i].get(v);
                m[v].A *= k;
                m[v].H = cut ? in : fmaf(k, m[v].H, in);
            }
        });
        if (RESET && s.cuts)
#pragma unroll
            for (int v = 0; v < VEC; v++) m[v].A = CUT;
        maps.put(P.wave, P.lane, m);
        __syncthreads();
        anew(Z);
        anew(x);
    } else {
        over_steps<STEPS, RESET, false>(s, [&](int i, bool) {
#pragma unroll
            for (int v = 0; v < VEC; v++) Z[i][v] = gate_of<E>(g[i].get(v));
        });
    }
#pragma unroll
    for (int v = 0; v < VEC; v++) h[v] = state && P.on ? state[P.b * S.D + P.d + v] : 0.0f;
    if constexpr (!ONE) {
        Map own = {1.0f, 0.0f};
        if (P.wave < VEC)
#pragma unroll
            for (int w = 0; w < WAVES; w++) own = then(own, maps.get(w, P.wave * WAVE + P.lane));
        before.wait(R, S, P.b, P.p, P.d0, P.wave, P.lane, own);
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VEC; v++) h[v] = before.from(h[v], P.lane, v);
    }
    if constexpr (WAVES > 1)
        for (int w = 0; w < P.wave; w++)
#pragma unroll
            for (int v = 0; v < VEC; v++) h[v] = apply(maps.get(w, P.lane * VEC + v), h[v]);
    const Rows<ONCE> to(out + P.b * S.T * S.D + P.d0, S.ot, s, width);
    over_steps<STEPS, RESET, false>(s, [&](int i, bool cut) {
        if (i % SPAN == 0 && carry && P.on && i < s.steps)
#pragma unroll
            for (int v = 0; v < VEC; v++) carry[(P.b * S.spans + (s.t0 + i) / SPAN) * S.D + P.d + v] = h[v];
        float o[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            float z, k;
            both(Z[i][v], z, k);
            const float in = z * x[i].get(v);
            h[v] = cut ? in : fmaf(k, h[v], in);
            o[v] = h[v];
        }
        to.template store<Word<E, VEC>::BYTES>(Word<E, VEC>::of(o).bits, i, at);
    });
    if (P.on && s.steps && s.t0 + s.steps == S.T)
#pragma unroll
        for (int v = 0; v < VEC; v++) last[P.b * S.D + P.d + v] = h[v];
}

template <typename E, int VEC, int STEPS, int WAVES, bool ONE, bool RESET, bool ONCE>
__global__ __launch_bounds__(WAVES* WAVE) __attribute__((amdgpu_waves_per_eu(VEC == 2 && WAVES > 1 ? 4 : 1))) void scan_back_kernel(Shape S, Records R, const E* __restrict__ gate, const E* __restrict__ value,
                                                                const uint8_t* __restrict__ reset, const float* __restrict__ carry,
                                                                const E* __restrict__ d_out, const float* __restrict__ d_last, E* __restrict__ d_gate,
                                                                E* __restrict__ d_value, float* __restrict__ d_state) {
    __shared__ Maps<VEC, WAVES> maps;
    __shared__ Before<VEC, WAVES> before;
    const Place<VEC, WAVES, ONE> P(S, R);
    const int64_t c = S.chunks - 1 - P.p;              // the walk begins at the last chunk
    const Span s = span_of<STEPS>(S, reset, P.b, (c * WAVES + P.wave) * STEPS, P.lane);
    const uint32_t at = P.on ? uint32_t(P.d - P.d0) * sizeof(E) : NO_LANE;
    const int64_t width = S.D - P.d0 < WAVE * VEC ? S.D - P.d0 : WAVE * VEC;
    Word<E, VEC> g[STEPS], x[STEPS], y[STEPS];
    load_steps(g, Rows<ONCE>(gate + P.b * S.gb + P.d0, S.gt, s, width), at);
    load_steps(x, Rows<ONCE>(value + P.b * S.vb + P.d0, S.vt, s, width), at);
    load_steps(y, Rows<ONCE>(d_out + P.b * S.db + P.d0, S.dt, s, width), at);
    end_steps(g, s, -INFINITY);
    end_steps(x, s, 0.0f);
    end_steps(y, s, 0.0f);
    float Z[STEPS][VEC], C[VEC], h[VEC];
    over_steps<STEPS, RESET, false>(s, [&](int i, bool) {
#pragma unroll
        for (int v = 0; v < VEC; v++) Z[i][v] = gate_of<E>(g[i].get(v));
    });
#pragma unroll
    for (int v = 0; v < VEC; v++) h[v] = P.on && s.steps ? carry[(P.b * S.spans + s.t0 / SPAN) * S.D + P.d + v] : 0.0f;
    if constexpr (WAVES > 1) {
        Map m[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) m[v] = {1.0f, 0.0f};
        over_steps<STEPS, RESET, true>(s, [&](int i, bool cut) {
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                float z, k;
                both(Z[i][v], z, k);
                m[v].A *= k;
                m[v].H = cut ? 0.0f : k * (y[i].get(v) + m[v].H);
            }
        });
        if (RESET && s.cuts)
#pragma unroll
            for (int v = 0; v < VEC; v++) m[v].A = CUT;
        maps.put(P.wave, P.lane, m);
        __syncthreads();
        anew(Z);
        anew(y);
    }
#pragma unroll
    for (int v = 0; v < VEC; v++) C[v] = d_last && P.on ? d_last[P.b * S.D + P.d + v] : 0.0f;
    if constexpr (!ONE) {
        Map own = {1.0f, 0.0f};
        if (P.wave < VEC)
#pragma unroll
            for (int w = WAVES - 1; w >= 0; w--) own = then(own, maps.get(w, P.wave * WAVE + P.lane));
        before.wait(R, S, P.b, P.p, P.d0, P.wave, P.lane, own);
    }
    float U[STEPS][VEC];                   // value minus the state before each step
    over_steps<STEPS, RESET, false>(s, [&](int i, bool cut) {
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            float z, k;
            both(Z[i][v], z, k);
            if (cut) h[v] = 0.0f;
            const float a = x[i].get(v);
            U[i][v] = a - h[v];
            h[v] = fmaf(k, h[v], z * a);
        }
    });
    if constexpr (!ONE) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VEC; v++) C[v] = before.from(C[v], P.lane, v);
    }
    if constexpr (WAVES > 1)
        for (int w = WAVES - 1; w > P.wave; w--)
#pragma unroll
            for (int v = 0; v < VEC; v++) C[v] = apply(maps.get(w, P.lane * VEC + v), C[v]);
    anew(Z);
    const Rows<ONCE> to_gate(d_gate + P.b * S.T * S.D + P.d0, S.ot, s, width), to_value(d_value + P.b * S.T * S.D + P.d0, S.ot, s, width);
    over_steps<STEPS, RESET, true>(s, [&](int i, bool cut) {
        float og[VEC], ov[VEC];
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            float z, k;
            both(Z[i][v], z, k);
            const float G = y[i].get(v) + C[v], in = z * G;
            ov[v] = in;
            og[v] = in * k * U[i][v];
            C[v] = cut ? 0.0f : k * G;
        }
        to_value.template store<Word<E, VEC>::BYTES>(Word<E, VEC>::of(ov).bits, i, at);
        to_gate.template store<Word<E, VEC>::BYTES>(Word<E, VEC>::of(og).bits, i, at);
    });
    if (d_state && P.on && c == 0 && P.wave == 0)
#pragma unroll
        for (int v = 0; v < VEC; v++) d_state[P.b * S.D + P.d + v] = C[v];
}

int64_t spans_of(int64_t T) { return (T + SPAN - 1) / SPAN; }
int64_t chunks_of(int64_t T, int steps) {
    const int64_t chunk = T <= steps ? steps : steps * CHUNK_WAVES;
    return (T + chunk - 1) / chunk;
}

// 8-byte words of a call's records: two for the counter, then the levels
int64_t words_of(int64_t B, int64_t chunks, int64_t D) {
    if (chunks <= 1) return 0;
    int64_t n = 2;
    for (; chunks; chunks /= FAN) n += B * chunks * D;
    return n;
}

// Channels of a lane, and tiles of D by waves of that many
int vec_of(int64_t D, int32_t dtype) { return element_bytes(dtype) == 2 && D > 1 ? 2 : 1; }
int64_t tiles_of(int64_t D, int vec) { return (D + WAVE * vec - 1) / (WAVE * vec); }

// What both entries ask of their arguments
template <int STEPS, typename... I> int32_t check(int64_t B, int64_t T, int64_t D, int32_t dtype, const void* work, uint64_t work_bytes, char* err, size_t cap, I... steps) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, cap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (B < 0 || T < 1 || D < 0) return fail(PV_EARG, err, cap, "shape: B >= 0, T >= 1, D >= 0");
    const int64_t most = int64_t(1) << 40;
    if (B > INT32_MAX || T > INT32_MAX || D > INT32_MAX || (B && D && (B * D > most || T > most / (B * D)))) return fail(PV_EARG, err, cap, "shape: B T D of 2^40 at most");
    const int64_t groups = B * chunks_of(T, STEPS) * tiles_of(D, vec_of(D, dtype)), items = (T <= STEPS ? 1 : CHUNK_WAVES) * WAVE;
    if (groups >= MOST_ITEMS / items) return fail(PV_EARG, err, cap, "shape: too many chunks for a launch's work items");
    for (int64_t st : {steps...}) if (T > 1 && (st < 0 || st * element_bytes(dtype) > MOST_STRIDE)) return fail(PV_EARG, err, cap, "stride: a step's is 0 to 2^26 bytes");
    const uint64_t need = pv_gated_scan_work_bytes(B, T, D);
    if (need && (!work || work_bytes < need || !aligned(work, 16))) return fail(PV_EARG, err, cap, "work: too small, or not 16-byte aligned");
    return PV_OK;
}

// Whether a call's accesses get the hint ONCE: tensors that the caches (256 MB) do not hold from one kernel to the next, with rows
// of whole 128-byte lines (of a line shared by two workgroups each would read it all). 8 x 8,192 x 1,024 (134 MB a tensor in
// bfloat16) 99 us forwards and 142 backwards with it, 105 and 156 without; 5 x 2,049 x 512 float32 (21 MB) 28 and 36 with it, 24
// and 33 without; 5 x 2,049 x 500, rows off the lines, 29 and 44, and 25 and 35.
bool once_of(int64_t B, int64_t T, int64_t D, int bytes) { return D * bytes % 128 == 0 && B * T * D * bytes >= (int64_t(64) << 20); }

// f(channels of a lane, steps of a wave, waves, one chunk only, resets, once) with the records cleared
template <int STEPS, typename F> int32_t launch(Shape& S, bool pairs, bool resets, bool once, void* work, hipStream_t st, F&& f) {
    // A single step's row may be longer than 32 bits hold: the steps that are not there are put where each access is behind the row's end
    if (S.T == 1) S.gt = S.vt = S.dt = S.ot = 2 * WAVE;
    S.spans = spans_of(S.T);
    S.chunks = chunks_of(S.T, STEPS);
    S.tiles = tiles_of(S.D, pairs ? 2 : 1);
    Records R = {};
    if (const int64_t words = words_of(S.B, S.chunks, S.D)) {
        uint64_t* w = static_cast<uint64_t*>(work);
        const int64_t need = (words + 1023) / 1024;
        records_kernel<<<uint32_t(need < 2048 ? need : 2048), 256, 0, st>>>(w, words);
        R.next = reinterpret_cast<uint32_t*>(w);
        w += 2;
        int64_t n = S.chunks;
        for (int l = 0; l < LEVELS; l++, n /= FAN) { R.level[l] = w; w += S.B * n * S.D; }
    }
    const uint32_t groups = uint32_t(S.B * S.tiles * S.chunks);
    using std::integral_constant;
    auto with = [&](auto vec, auto resets) {
        const integral_constant<int, STEPS> steps;
        const integral_constant<int, CHUNK_WAVES> waves;
        if constexpr (STEPS > STEPS_BACK)
            if (S.T <= STEPS_SHORT) return f(vec, integral_constant<int, STEPS_SHORT>{}, integral_constant<int, 1>{}, std::true_type{}, resets, std::false_type{}, R, groups);
        if (S.T <= STEPS) return f(vec, steps, integral_constant<int, 1>{}, std::true_type{}, resets, std::false_type{}, R, groups);
        if (S.chunks == 1) return f(vec, steps, waves, std::true_type{}, resets, std::false_type{}, R, groups);
        if (once) return f(vec, steps, waves, std::false_type{}, resets, std::true_type{}, R, groups);
        return f(vec, steps, waves, std::false_type{}, resets, std::false_type{}, R, groups);
    };
    if (pairs) return resets ? with(integral_constant<int, 2>{}, std::true_type{}) : with(integral_constant<int, 2>{}, std::false_type{});
    return resets ? with(integral_constant<int, 1>{}, std::true_type{}) : with(integral_constant<int, 1>{}, std::false_type{});
}

}  // namespace

extern "C" {

int64_t pv_gated_scan_spans(int64_t T) { return T > 0 ? spans_of(T) : 0; }
uint64_t pv_gated_scan_work_bytes(int64_t B, int64_t T, int64_t D) {
    return B > 0 && T > 0 && D > 0 ? uint64_t(words_of(B, chunks_of(T, STEPS_BACK), D)) * 8 : 0;
}

int32_t pv_gated_scan_hip(const void* gate, const void* value, const float* state, const uint8_t* reset, int64_t B, int64_t T, int64_t D, int64_t gate_b,
                          int64_t gate_t, int64_t value_b, int64_t value_t, int32_t dtype, void* out, float* last, float* carry, void* work,
                          uint64_t work_bytes, void* stream, char* err, size_t errcap) {
    if (int32_t e = check<STEPS_FORWARD>(B, T, D, dtype, work, work_bytes, err, errcap, gate_t, value_t, D)) return e;
    if (!B || !D) return PV_OK;
    if (!gate || !value || !out || !last) return fail(PV_EARG, err, errcap, "null argument");
    Shape S{B, T, D, gate_b, gate_t, value_b, value_t, 0, 0, D, 0, 0, 0};
    const hipStream_t st = hipStream_t(stream);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        const bool pairs = vec_of(D, dtype) == 2;
        return launch<STEPS_FORWARD>(S, pairs, reset, once_of(B, T, D, sizeof(E)), work, st, [&](auto vec, auto steps, auto waves, auto one, auto resets, auto once, const Records& R, uint32_t groups) {
            constexpr int V = decltype(vec)::value, N = decltype(steps)::value, W = decltype(waves)::value;
            constexpr bool ONE = decltype(one)::value, RESET = decltype(resets)::value, ONCE = decltype(once)::value && V * sizeof(E) == 4;
            if constexpr (V == 1 || sizeof(E) == 2)
                scan_kernel<E, V, N, W, ONE, RESET, ONCE><<<groups, W * WAVE, 0, st>>>(S, R, static_cast<const E*>(gate), static_cast<const E*>(value), state, reset,
                                                                       static_cast<E*>(out), last, carry);
            return launched(err, errcap);
        });
    });
}

int32_t pv_gated_scan_backward_hip(const void* gate, const void* value, const float* carry, const uint8_t* reset, int64_t B, int64_t T, int64_t D,
                                   int64_t gate_b, int64_t gate_t, int64_t value_b, int64_t value_t, const void* d_out, int64_t d_out_b, int64_t d_out_t,
                                   const float* d_last, int32_t dtype, void* d_gate, void* d_value, float* d_state, void* work, uint64_t work_bytes,
                                   void* stream, char* err, size_t errcap) {
    if (int32_t e = check<STEPS_BACK>(B, T, D, dtype, work, work_bytes, err, errcap, gate_t, value_t, d_out_t, D)) return e;
    if (!B || !D) return PV_OK;
    if (!gate || !value || !carry || !d_out || !d_gate || !d_value) return fail(PV_EARG, err, errcap, "null argument");
    Shape S{B, T, D, gate_b, gate_t, value_b, value_t, d_out_b, d_out_t, D, 0, 0, 0};
    const hipStream_t st = hipStream_t(stream);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        const bool pairs = vec_of(D, dtype) == 2;
        return launch<STEPS_BACK>(S, pairs, reset, once_of(B, T, D, sizeof(E)), work, st, [&](auto vec, auto steps, auto waves, auto one, auto resets, auto once, const Records& R, uint32_t groups) {
            constexpr int V = decltype(vec)::value, N = decltype(steps)::value, W = decltype(waves)::value;
            constexpr bool ONE = decltype(one)::value, RESET = decltype(resets)::value, ONCE = decltype(once)::value && V * sizeof(E) == 4;
            if constexpr (V == 1 || sizeof(E) == 2)
                scan_back_kernel<E, V, N, W, ONE, RESET, ONCE><<<groups, W * WAVE, 0, st>>>(S, R, static_cast<const E*>(gate), static_cast<const E*>(value), reset, carry,
                                                                            static_cast<const E*>(d_out), d_last, static_cast<E*>(d_gate),
                                                                            static_cast<E*>(d_value), d_state);
            return launched(err, errcap);
        });
    });
}

}  // extern "C"
