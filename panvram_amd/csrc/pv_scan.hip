// Gated linear recurrence h[t] = (1 - z[t]) h[t-1] + z[t] value[t], z = sigmoid(gate), over [B, T, D], and its gradients.
//
// A run of steps is the map h -> A h + H of the state before it: A the product of its (1 - z), H the run started at zero.
// Maps of neighbouring runs join, so all of T is worked on at once and every byte is read once and written once:
//   - a wave holds STEPS steps of 64 x VEC channels in registers, a workgroup of WAVES waves a chunk of WAVES x STEPS steps;
//   - the workgroup makes its chunk's map, publishes it (`before_chunk`), joins the maps of the chunks before, and walks its
//     steps from there.
// The gradient is the same recurrence backwards: C[t] = (1 - z[t]) (d_out[t] + C[t+1]), C what flows into h[t-1]; the states
// before each step are made again from the chunk's start, which the forward pass leaves in `carry` (one f32 per chunk and
// channel, so that h is never read). A step's arithmetic is the same for every cut of T, and so is the order in which maps are
// joined: results do not depend on which workgroup was faster.
//
// A reset at t drops h[t-1], whatever it holds (a NaN too): the step is chosen, not multiplied by zero, and the map of a run
// with a reset in it has A = CUT, which no product of (1 - z) can be.
#include "pv_ops.h"

using namespace pvo;

namespace {

constexpr int STEPS = 16;                  // of a wave: 16 loads of each tensor in flight
constexpr int CHUNK_WAVES = 8;             // of a workgroup, where T has more than STEPS steps
constexpr float CUT = -1.0f;

struct Shape {
    int64_t B, T, D, gb, gt, vb, vt, db, dt;   // strides in elements: gate, value, d_out (batch, time); channels are neighbours
    int64_t chunks, tiles;                     // chunks of T, tiles of D
};

// z = sigmoid(g) and 1 - z, each to a few units in its last place: from exp(-|g|), so that neither is a difference
__device__ inline void sigmoid2(float g, float& z, float& keep) {
    const float e = __expf(-fabsf(g));
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    const float s = e * r;
    z = g >= 0.0f ? r : s;
    keep = g >= 0.0f ? s : r;
}

template <int VEC> struct Map { float A[VEC], H[VEC]; };
template <int VEC> __device__ inline Map<VEC> identity() {
    Map<VEC> m;
#pragma unroll
    for (int v = 0; v < VEC; v++) { m.A[v] = 1.0f; m.H[v] = 0.0f; }
    return m;
}
__device__ inline float apply(float A, float H, float before) { return A == CUT ? H : fmaf(A, before, H); }
template <int VEC> __device__ inline Map<VEC> then(const Map<VEC>& first, const Map<VEC>& second) {
    Map<VEC> m;
#pragma unroll
    for (int v = 0; v < VEC; v++) {
        m.H[v] = apply(second.A[v], second.H[v], first.H[v]);
        m.A[v] = first.A[v] == CUT || second.A[v] == CUT ? CUT : first.A[v] * second.A[v];
    }
    return m;
}

// ---- Maps of chunks, in the order of the walk (position 0 first), passed between workgroups.
// Level 0 has a map for each chunk, level l + 1 one for each FAN whole neighbours of level l. The workgroup at position p needs
// the maps of its predecessors within its group of FAN, of their group's predecessors within its, and so on: the base-FAN
// digits of p, at most FAN - 1 maps a level. The last of a group makes the group's map of them and its own.
//
// A map is one 8-byte word (A, H) per channel, written by one store; EMPTY until then. Its NaNs are stored as 0x7fc00000, so
// that no map is EMPTY. A word is read and written past the L2 caches (agent scope); no other data depends on the order.
// Every wait ends: a workgroup takes its position from a counter, so all earlier positions belong to workgroups that run
// already, a position publishes level 0 without waiting, and each level waits for earlier positions only. (Should a word not
// come in some seconds all the same, it counts as NaN.)
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
template <int VEC> __device__ inline void publish(uint64_t* at, const Map<VEC>& m, bool on) {
    if (!on) return;
#pragma unroll
    for (int v = 0; v < VEC; v++) __hip_atomic_store(at + v, word_of(m.A[v], m.H[v]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The map of all chunks before position p, for one wave's channels (from d on, where `on`); own: the chunk's map
template <int VEC> __device__ inline Map<VEC> before_chunk(const Records& R, const Shape& S, int64_t b, int64_t p, int64_t d, bool on, Map<VEC> own) {
    Map<VEC> all = identity<VEC>();
    int64_t n = S.chunks;
    bool whole = true;                     // own is the map of a whole group of this level
    for (int l = 0; l < LEVELS && n > 0; l++, n /= FAN) {
        const int64_t at = p & ~int64_t(FAN - 1);      // the group's first
        const int many = int(p - at);
        uint64_t* rec = R.level[l] + b * n * S.D + d;
        if (whole) publish<VEC>(rec + p * S.D, own, on);
        uint64_t w[FAN - 1][VEC];
#pragma unroll
        for (int i = 0; i < FAN - 1; i++)
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                w[i][v] = 0;
                if (i < many && on) w[i][v] = __hip_atomic_load(rec + (at + i) * S.D + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        Map<VEC> level = identity<VEC>();
#pragma unroll
        for (int i = 0; i < FAN - 1; i++) {
            if (i >= many) break;
            Map<VEC> m;
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                for (int k = 0; __any(w[i][v] == EMPTY) && k < POLLS; k++) {
                    __builtin_amdgcn_s_sleep(1);
                    if (on) w[i][v] = __hip_atomic_load(rec + (at + i) * S.D + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
                m.A[v] = __uint_as_float(uint32_t(w[i][v]));
                m.H[v] = __uint_as_float(uint32_t(w[i][v] >> 32));
            }
            level = then(level, m);
        }
        all = then(level, all);
        whole = whole && many == FAN - 1;
        if (whole) own = then(level, own);
        p /= FAN;
    }
    return all;
}

// ---- What a workgroup works on: channels d.. of sequence b, position p of the walk
template <int VEC, int WAVES, bool ONE> struct Place {
    int64_t b, p, d0, d;                   // d: the lane's first channel, d0: the wave's
    uint32_t at;                           // d - d0
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
        p = turn / rows;
        const uint32_t rest = turn % rows;
        b = rest / uint32_t(S.tiles);
        d0 = int64_t(rest % uint32_t(S.tiles)) * (WAVE * VEC);
        at = uint32_t(lane * VEC);
        d = d0 + at;
        on = d < S.D;
    }
};

// A wave's steps [t0, t0 + steps), and a bit for each that has a reset
struct Span { int64_t t0; int steps; uint32_t cuts; };
__device__ inline Span span_of(const Shape& S, const uint8_t* reset, int64_t b, int64_t t0, int lane) {
    Span s;
    s.t0 = t0;
    const int64_t left = S.T - t0;
    s.steps = left <= 0 ? 0 : left < STEPS ? int(left) : STEPS;
    s.cuts = 0;
    if (reset) s.cuts = uint32_t(__ballot(lane < s.steps && reset[b * S.T + t0 + lane] != 0));
    return s;
}
// (from is the same for the wave, at: the lane's channel in it)
template <typename E, int VEC> __device__ inline void load_steps(pack<E, VEC>* to, const E* from, int64_t stride, const Span& s, uint32_t at, bool on) {
    from += s.t0 * stride;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        if (on && i < s.steps) to[i] = pack<E, VEC>::load(from + i * stride + at);
        else
#pragma unroll
            for (int v = 0; v < VEC; v++) to[i].v[v] = E(0.0f);
    }
}

template <typename E, int VEC, int WAVES, bool ONE>
__global__ __launch_bounds__(WAVES* WAVE) void scan_kernel(Shape S, Records R, const E* __restrict__ gate, const E* __restrict__ value,
                                                           const float* __restrict__ state, const uint8_t* __restrict__ reset, E* __restrict__ out,
                                                           float* __restrict__ last, float* __restrict__ carry) {
    __shared__ Map<VEC> maps[WAVES][WAVE];
    __shared__ float starts[VEC][WAVE];
    const Place<VEC, WAVES, ONE> P(S, R);
    const Span s = span_of(S, reset, P.b, (P.p * WAVES + P.wave) * STEPS, P.lane);
    pack<E, VEC> g[STEPS], x[STEPS];
    load_steps<E, VEC>(g, gate + P.b * S.gb + P.d0, S.gt, s, P.at, P.on);
    load_steps<E, VEC>(x, value + P.b * S.vb + P.d0, S.vt, s, P.at, P.on);
    float K[STEPS][VEC], X[STEPS][VEC];
    Map<VEC> m = identity<VEC>();
#pragma unroll
    for (int i = 0; i < STEPS; i++)
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            float z;
            sigmoid2(float(g[i].v[v]), z, K[i][v]);
            X[i][v] = z * float(x[i].v[v]);
            if (i >= s.steps) { K[i][v] = 1.0f; X[i][v] = 0.0f; }
            m.A[v] *= K[i][v];
            m.H[v] = s.cuts >> i & 1 ? X[i][v] : fmaf(K[i][v], m.H[v], X[i][v]);
        }
    if (s.cuts)
#pragma unroll
        for (int v = 0; v < VEC; v++) m.A[v] = CUT;
    if constexpr (WAVES > 1) {
        maps[P.wave][P.lane] = m;
        __syncthreads();
    }
    float h[VEC];
    if (ONE || P.wave == 0) {
#pragma unroll
        for (int v = 0; v < VEC; v++) h[v] = state && P.on ? state[P.b * S.D + P.d + v] : 0.0f;
    }
    if (P.wave == 0) {
        if constexpr (!ONE) {
            Map<VEC> own = m;
#pragma unroll
            for (int w = 1; w < WAVES; w++) own = then(own, maps[w][P.lane]);
            const Map<VEC> b = before_chunk<VEC>(R, S, P.b, P.p, P.d, P.on, own);
#pragma unroll
            for (int v = 0; v < VEC; v++) starts[v][P.lane] = h[v] = apply(b.A[v], b.H[v], h[v]);
        }
        if (carry && P.on)
#pragma unroll
            for (int v = 0; v < VEC; v++) carry[(P.b * S.chunks + P.p) * S.D + P.d + v] = h[v];
    }
    if constexpr (!ONE) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VEC; v++) h[v] = starts[v][P.lane];
    }
    for (int w = 0; w < P.wave; w++)
#pragma unroll
        for (int v = 0; v < VEC; v++) h[v] = apply(maps[w][P.lane].A[v], maps[w][P.lane].H[v], h[v]);
    E* to = out + (P.b * S.T + s.t0) * S.D + P.d0;
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        pack<E, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            h[v] = s.cuts >> i & 1 ? X[i][v] : fmaf(K[i][v], h[v], X[i][v]);
            o.v[v] = E(h[v]);
        }
        if (P.on && i < s.steps) o.store(to + i * S.D + P.at);
    }
    if (P.on && s.steps && s.t0 + s.steps == S.T)
#pragma unroll
        for (int v = 0; v < VEC; v++) last[P.b * S.D + P.d + v] = h[v];
}

template <typename E, int VEC, int WAVES, bool ONE>
__global__ __launch_bounds__(WAVES* WAVE) void scan_back_kernel(Shape S, Records R, const E* __restrict__ gate, const E* __restrict__ value,
                                                                const uint8_t* __restrict__ reset, const float* __restrict__ carry,
                                                                const E* __restrict__ d_out, const float* __restrict__ d_last, E* __restrict__ d_gate,
                                                                E* __restrict__ d_value, float* __restrict__ d_state) {
    __shared__ Map<VEC> maps[WAVES][WAVE];             // forwards: (A, H); backwards: (A, flows)
    __shared__ float flows[WAVES][VEC][WAVE], ends[VEC][WAVE];
    const Place<VEC, WAVES, ONE> P(S, R);
    const int64_t c = S.chunks - 1 - P.p;              // the walk begins at the last chunk
    const Span s = span_of(S, reset, P.b, (c * WAVES + P.wave) * STEPS, P.lane);
    pack<E, VEC> g[STEPS], x[STEPS], y[STEPS];
    load_steps<E, VEC>(g, gate + P.b * S.gb + P.d0, S.gt, s, P.at, P.on);
    load_steps<E, VEC>(x, value + P.b * S.vb + P.d0, S.vt, s, P.at, P.on);
    load_steps<E, VEC>(y, d_out + P.b * S.db + P.d0, S.dt, s, P.at, P.on);
    // z and 1 - z of a step in one register: the smaller of the two, its sign bit set where that is z. The other is 1 minus it,
    // at least a half and so as exact.
    float Z[STEPS][VEC];
    auto both = [&](float q, float& z, float& k) {
        const float a = fabsf(q), b = 1.0f - a;
        const bool low = int32_t(__float_as_uint(q)) < 0;
        z = low ? a : b;
        k = low ? b : a;
    };
    Map<VEC> m = identity<VEC>();
#pragma unroll
    for (int i = 0; i < STEPS; i++)
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const float a = float(g[i].v[v]), e = __expf(-fabsf(a));
            const float q = i < s.steps ? copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), a) : -0.0f;
            Z[i][v] = q;
            float z, k;
            both(q, z, k);
            const float in = z * float(x[i].v[v]);
            m.A[v] *= k;
            m.H[v] = s.cuts >> i & 1 ? in : fmaf(k, m.H[v], in);
        }
    float C[VEC] = {};
#pragma unroll
    for (int i = STEPS - 1; i >= 0; i--)
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            float z, k;
            both(Z[i][v], z, k);
            C[v] = s.cuts >> i & 1 ? 0.0f : k * (float(y[i].v[v]) + C[v]);
        }
    if (s.cuts)
#pragma unroll
        for (int v = 0; v < VEC; v++) m.A[v] = CUT;
    if constexpr (WAVES > 1) {
        maps[P.wave][P.lane] = m;
#pragma unroll
        for (int v = 0; v < VEC; v++) flows[P.wave][v][P.lane] = C[v];
        __syncthreads();
    }
    float end[VEC];
    if (ONE || P.wave == 0) {
#pragma unroll
        for (int v = 0; v < VEC; v++) end[v] = d_last && P.on ? d_last[P.b * S.D + P.d + v] : 0.0f;
    }
    if constexpr (!ONE) {
        if (P.wave == 0) {
            Map<VEC> own = identity<VEC>();
#pragma unroll
            for (int w = WAVES - 1; w >= 0; w--) {
                Map<VEC> k = maps[w][P.lane];
#pragma unroll
                for (int v = 0; v < VEC; v++) k.H[v] = flows[w][v][P.lane];
                own = then(own, k);
            }
            const Map<VEC> b = before_chunk<VEC>(R, S, P.b, P.p, P.d, P.on, own);
#pragma unroll
            for (int v = 0; v < VEC; v++) ends[v][P.lane] = apply(b.A[v], b.H[v], end[v]);
        }
    }
    // value minus the state before each step
    float h[VEC], U[STEPS][VEC];
#pragma unroll
    for (int v = 0; v < VEC; v++) h[v] = P.on ? carry[(P.b * S.chunks + c) * S.D + P.d + v] : 0.0f;
    for (int w = 0; w < P.wave; w++)
#pragma unroll
        for (int v = 0; v < VEC; v++) h[v] = apply(maps[w][P.lane].A[v], maps[w][P.lane].H[v], h[v]);
#pragma unroll
    for (int i = 0; i < STEPS; i++)
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            float z, k;
            both(Z[i][v], z, k);
            if (s.cuts >> i & 1) h[v] = 0.0f;
            const float a = float(x[i].v[v]);
            U[i][v] = a - h[v];
            h[v] = fmaf(k, h[v], z * a);
        }
    if constexpr (!ONE) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VEC; v++) end[v] = ends[v][P.lane];
    }
#pragma unroll
    for (int v = 0; v < VEC; v++) C[v] = end[v];
    for (int w = WAVES - 1; w > P.wave; w--)
#pragma unroll
        for (int v = 0; v < VEC; v++) C[v] = apply(maps[w][P.lane].A[v], flows[w][v][P.lane], C[v]);
    E* const to_gate = d_gate + (P.b * S.T + s.t0) * S.D + P.d0;
    E* const to_value = d_value + (P.b * S.T + s.t0) * S.D + P.d0;
#pragma unroll
    for (int i = STEPS - 1; i >= 0; i--) {
        pack<E, VEC> og, ov;
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            float z, k;
            both(Z[i][v], z, k);
            const float G = float(y[i].v[v]) + C[v], in = z * G;
            ov.v[v] = E(in);
            og.v[v] = E(in * k * U[i][v]);
            C[v] = s.cuts >> i & 1 ? 0.0f : k * G;
        }
        if (P.on && i < s.steps) {
            ov.store(to_value + i * S.D + P.at);
            og.store(to_gate + i * S.D + P.at);
        }
    }
    if (d_state && P.on && c == 0 && P.wave == 0)
#pragma unroll
        for (int v = 0; v < VEC; v++) d_state[P.b * S.D + P.d + v] = C[v];
}

int64_t chunk_steps(int64_t T) { return T <= STEPS ? STEPS : STEPS * CHUNK_WAVES; }
int64_t chunks_of(int64_t T) { return (T + chunk_steps(T) - 1) / chunk_steps(T); }

// 8-byte words of a call's records: two for the counter, then the levels
int64_t words_of(int64_t B, int64_t chunks, int64_t D) {
    if (chunks <= 1) return 0;
    int64_t n = 2;
    for (; chunks; chunks /= FAN) n += B * chunks * D;
    return n;
}

// What both entries ask of their arguments
int32_t check(int64_t B, int64_t T, int64_t D, int32_t dtype, const void* work, uint64_t work_bytes, char* err, size_t cap) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, cap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (B < 0 || T < 1 || D < 0) return fail(PV_EARG, err, cap, "shape: B >= 0, T >= 1, D >= 0");
    const int64_t most = int64_t(1) << 40;
    if (B > INT32_MAX || T > INT32_MAX || D > INT32_MAX || (B && D && (B * D > most || T > most / (B * D)))) return fail(PV_EARG, err, cap, "shape: B T D of 2^40 at most");
    if (B && D && B * chunks_of(T) * ((D + WAVE - 1) / WAVE) > INT32_MAX) return fail(PV_EARG, err, cap, "shape: too many chunks");
    const uint64_t need = pv_gated_scan_work_bytes(B, T, D);
    if (need && (!work || work_bytes < need || !aligned(work, 16))) return fail(PV_EARG, err, cap, "work: too small, or not 16-byte aligned");
    return PV_OK;
}

// f(vector of channels, waves, one chunk only) with the records cleared
template <typename F> int32_t launch(Shape& S, bool pairs, void* work, hipStream_t st, F&& f) {
    const int vec = pairs ? 2 : 1;
    S.chunks = chunks_of(S.T);
    S.tiles = (S.D + WAVE * vec - 1) / (WAVE * vec);
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
    auto with = [&](auto vec) {
        if (S.T <= STEPS) return f(vec, integral_constant<int, 1>{}, integral_constant<bool, true>{}, R, groups);
        if (S.chunks == 1) return f(vec, integral_constant<int, CHUNK_WAVES>{}, integral_constant<bool, true>{}, R, groups);
        return f(vec, integral_constant<int, CHUNK_WAVES>{}, integral_constant<bool, false>{}, R, groups);
    };
    return pairs ? with(integral_constant<int, 2>{}) : with(integral_constant<int, 1>{});
}

// Whether a [B, T, D] tensor's rows can be read two channels at a time
template <typename E> bool pairs_of(const void* p, int64_t B, int64_t T, int64_t sb, int64_t st) {
    return aligned(p, 2 * sizeof(E)) && (B == 1 || sb % 2 == 0) && (T == 1 || st % 2 == 0);
}

}  // namespace

extern "C" {

int64_t pv_gated_scan_chunks(int64_t T) { return T > 0 ? chunks_of(T) : 0; }
uint64_t pv_gated_scan_work_bytes(int64_t B, int64_t T, int64_t D) {
    return B > 0 && T > 0 && D > 0 ? uint64_t(words_of(B, chunks_of(T), D)) * 8 : 0;
}

int32_t pv_gated_scan_hip(const void* gate, const void* value, const float* state, const uint8_t* reset, int64_t B, int64_t T, int64_t D, int64_t gate_b,
                          int64_t gate_t, int64_t value_b, int64_t value_t, int32_t dtype, void* out, float* last, float* carry, void* work,
                          uint64_t work_bytes, void* stream, char* err, size_t errcap) {
    if (int32_t e = check(B, T, D, dtype, work, work_bytes, err, errcap)) return e;
    if (!B || !D) return PV_OK;
    if (!gate || !value || !out || !last) return fail(PV_EARG, err, errcap, "null argument");
    Shape S{B, T, D, gate_b, gate_t, value_b, value_t, 0, 0, 0, 0};
    const hipStream_t st = hipStream_t(stream);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        const bool pairs = sizeof(E) == 2 && D % 2 == 0 && pairs_of<E>(gate, B, T, gate_b, gate_t) && pairs_of<E>(value, B, T, value_b, value_t) && aligned(out, 4);
        return launch(S, pairs, work, st, [&](auto vec, auto waves, auto one, const Records& R, uint32_t groups) {
            constexpr int V = decltype(vec)::value, W = decltype(waves)::value;
            constexpr bool ONE = decltype(one)::value;
            if constexpr (V == 1 || sizeof(E) == 2)
                scan_kernel<E, V, W, ONE><<<groups, W * WAVE, 0, st>>>(S, R, static_cast<const E*>(gate), static_cast<const E*>(value), state, reset,
                                                                       static_cast<E*>(out), last, carry);
            return launched(err, errcap);
        });
    });
}

int32_t pv_gated_scan_backward_hip(const void* gate, const void* value, const float* carry, const uint8_t* reset, int64_t B, int64_t T, int64_t D,
                                   int64_t gate_b, int64_t gate_t, int64_t value_b, int64_t value_t, const void* d_out, int64_t d_out_b, int64_t d_out_t,
                                   const float* d_last, int32_t dtype, void* d_gate, void* d_value, float* d_state, void* work, uint64_t work_bytes,
                                   void* stream, char* err, size_t errcap) {
    if (int32_t e = check(B, T, D, dtype, work, work_bytes, err, errcap)) return e;
    if (!B || !D) return PV_OK;
    if (!gate || !value || !carry || !d_out || !d_gate || !d_value) return fail(PV_EARG, err, errcap, "null argument");
    Shape S{B, T, D, gate_b, gate_t, value_b, value_t, d_out_b, d_out_t, 0, 0};
    const hipStream_t st = hipStream_t(stream);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        const bool pairs = sizeof(E) == 2 && D % 2 == 0 && pairs_of<E>(gate, B, T, gate_b, gate_t) && pairs_of<E>(value, B, T, value_b, value_t) &&
                           pairs_of<E>(d_out, B, T, d_out_b, d_out_t) && aligned(d_gate, 4) && aligned(d_value, 4);
        return launch(S, pairs, work, st, [&](auto vec, auto waves, auto one, const Records& R, uint32_t groups) {
            constexpr int V = decltype(vec)::value, W = decltype(waves)::value;
            constexpr bool ONE = decltype(one)::value;
            if constexpr (V == 1 || sizeof(E) == 2)
                scan_back_kernel<E, V, W, ONE><<<groups, W * WAVE, 0, st>>>(S, R, static_cast<const E*>(gate), static_cast<const E*>(value), reset, carry,
                                                                            static_cast<const E*>(d_out), d_last, static_cast<E*>(d_gate),
                                                                            static_cast<E*>(d_value), d_state);
            return launched(err, errcap);
        });
    });
}

}  // extern "C"
