// Gated linear recurrence h[t] = (1 - z[t]) h[t-1] + z[t] value[t], z = sigmoid(gate), over [B, T, D], and its gradients.
//
// A run of steps is the map h -> A h + H of the state before it: A the product of its (1 - z), H the run started at zero.
// Maps of neighbouring runs join, so T is cut into chunks of CHUNK steps: one pass makes every chunk's map, a second walks
// the chunks' maps from the given state (each chunk's start state is `carry`), a third does the chunks from their starts.
// The gradient is the same recurrence backwards: C[t] = (1 - z[t]) (d_out[t] + C[t+1]), C what flows into h[t-1].
//
// A reset at t drops h[t-1], whatever it holds (a NaN too): the step is chosen, not multiplied by zero, and the map of a run
// with a reset in it has A = CUT, which no product of (1 - z) can be.
#include "pv_ops.h"

using namespace pvo;

namespace {

constexpr int CHUNK = 64;                  // steps of a chunk
constexpr int BLOCK = 256;                 // lanes of a workgroup, one channel each
constexpr float CUT = -1.0f;

// z = sigmoid(g) and 1 - z, each to a few units in its last place: from exp(-|g|), so that neither is a difference
__device__ inline void sigmoid2(float g, float& z, float& keep) {
    const float e = __expf(-fabsf(g));
    const float r = __builtin_amdgcn_rcpf(1.0f + e);
    const float s = e * r;
    z = g >= 0.0f ? r : s;
    keep = g >= 0.0f ? s : r;
}
__device__ inline float join(float A, float H, float before) { return A == CUT ? H : fmaf(A, before, H); }

struct Shape {
    int64_t B, T, D, gb, gt, vb, vt, db, dt;   // strides in elements: gate, value, d_out (batch, time); channels are neighbours
    int64_t chunks;
};

// What one lane works on: channel d of sequence b, steps [t0, t1)
struct Place { int64_t b, c, d, t0, t1; bool on; };
__device__ inline Place place(const Shape& S) {
    Place p;
    p.d = int64_t(blockIdx.x) * BLOCK + threadIdx.x;
    p.c = blockIdx.y;
    p.b = blockIdx.z;
    p.t0 = p.c * CHUNK;
    p.t1 = p.t0 + CHUNK < S.T ? p.t0 + CHUNK : S.T;
    p.on = p.d < S.D;
    return p;
}

template <typename E> __global__ __launch_bounds__(BLOCK) void scan_map_kernel(Shape S, const E* gate, const E* value, const uint8_t* reset, float2* maps) {
    const Place p = place(S);
    if (!p.on) return;
    float A = 1.0f, H = 0.0f;
    for (int64_t t = p.t0; t < p.t1; t++) {
        float z, k;
        sigmoid2(float(gate[p.b * S.gb + t * S.gt + p.d]), z, k);
        const float x = z * float(value[p.b * S.vb + t * S.vt + p.d]);
        if (reset && reset[p.b * S.T + t]) { A = CUT; H = x; }
        else { A = A == CUT ? CUT : A * k; H = fmaf(k, H, x); }
    }
    maps[(p.b * S.chunks + p.c) * S.D + p.d] = make_float2(A, H);
}

// carry[b, c, d]: the state before chunk c
__global__ __launch_bounds__(BLOCK) void scan_carry_kernel(Shape S, const float2* maps, const float* state, float* carry) {
    const int64_t d = int64_t(blockIdx.x) * BLOCK + threadIdx.x, b = blockIdx.y;
    if (d >= S.D) return;
    float h = state ? state[b * S.D + d] : 0.0f;
    for (int64_t c = 0; c < S.chunks; c++) {
        const int64_t i = (b * S.chunks + c) * S.D + d;
        carry[i] = h;
        h = join(maps[i].x, maps[i].y, h);
    }
}

template <typename E> __global__ __launch_bounds__(BLOCK)
void scan_apply_kernel(Shape S, const E* gate, const E* value, const uint8_t* reset, const float* carry, E* out, float* last) {
    const Place p = place(S);
    if (!p.on) return;
    float h = carry[(p.b * S.chunks + p.c) * S.D + p.d];
    for (int64_t t = p.t0; t < p.t1; t++) {
        float z, k;
        sigmoid2(float(gate[p.b * S.gb + t * S.gt + p.d]), z, k);
        const float x = z * float(value[p.b * S.vb + t * S.vt + p.d]);
        h = reset && reset[p.b * S.T + t] ? x : fmaf(k, h, x);
        out[(p.b * S.T + t) * S.D + p.d] = E(h);
    }
    if (p.t1 == S.T) last[p.b * S.D + p.d] = h;
}

// The backward map of a chunk: what flows out of its first step's h[t-1] from what flows into its last step's h[t]
template <typename E> __global__ __launch_bounds__(BLOCK) void scan_back_map_kernel(Shape S, const E* gate, const E* d_out, const uint8_t* reset, float2* maps) {
    const Place p = place(S);
    if (!p.on) return;
    float A = 1.0f, C = 0.0f;
    for (int64_t t = p.t1 - 1; t >= p.t0; t--) {
        float z, k;
        sigmoid2(float(gate[p.b * S.gb + t * S.gt + p.d]), z, k);
        if (reset && reset[p.b * S.T + t]) { A = CUT; C = 0.0f; }
        else { A = A == CUT ? CUT : A * k; C = k * (float(d_out[p.b * S.db + t * S.dt + p.d]) + C); }
    }
    maps[(p.b * S.chunks + p.c) * S.D + p.d] = make_float2(A, C);
}

// flow[b, c, d]: what flows into the last h of chunk c from behind it
__global__ __launch_bounds__(BLOCK) void scan_back_carry_kernel(Shape S, const float2* maps, const float* d_last, float* flow) {
    const int64_t d = int64_t(blockIdx.x) * BLOCK + threadIdx.x, b = blockIdx.y;
    if (d >= S.D) return;
    float C = d_last ? d_last[b * S.D + d] : 0.0f;
    for (int64_t c = S.chunks - 1; c >= 0; c--) {
        const int64_t i = (b * S.chunks + c) * S.D + d;
        flow[i] = C;
        C = join(maps[i].x, maps[i].y, C);
    }
}

template <typename E> __global__ __launch_bounds__(BLOCK)
void scan_back_apply_kernel(Shape S, const E* gate, const E* value, const uint8_t* reset, const float* carry, const float* flow, const E* d_out,
                            E* d_gate, E* d_value, float* d_state) {
    const Place p = place(S);
    if (!p.on) return;
    const int64_t at = (p.b * S.chunks + p.c) * S.D + p.d;
    // the states before each step, made again from the chunk's start
    float before[CHUNK];
    float h = carry[at];
#pragma unroll
    for (int i = 0; i < CHUNK; i++) {
        const int64_t t = p.t0 + i;
        if (t < p.t1) {
            float z, k;
            sigmoid2(float(gate[p.b * S.gb + t * S.gt + p.d]), z, k);
            if (reset && reset[p.b * S.T + t]) h = 0.0f;
            before[i] = h;
            h = fmaf(k, h, z * float(value[p.b * S.vb + t * S.vt + p.d]));
        }
    }
    float C = flow[at];
#pragma unroll
    for (int i = CHUNK - 1; i >= 0; i--) {
        const int64_t t = p.t0 + i;
        if (t < p.t1) {
            float z, k;
            sigmoid2(float(gate[p.b * S.gb + t * S.gt + p.d]), z, k);
            const float G = float(d_out[p.b * S.db + t * S.dt + p.d]) + C;
            const int64_t o = (p.b * S.T + t) * S.D + p.d;
            d_value[o] = E(z * G);
            d_gate[o] = E(z * k * G * (float(value[p.b * S.vb + t * S.vt + p.d]) - before[i]));
            C = reset && reset[p.b * S.T + t] ? 0.0f : k * G;
        }
    }
    if (d_state && p.c == 0) d_state[p.b * S.D + p.d] = C;
}

int64_t chunks_of(int64_t T) { return (T + CHUNK - 1) / CHUNK; }

// What both entries ask of their arguments
int32_t check(int64_t B, int64_t T, int64_t D, int32_t dtype, const void* work, uint64_t work_bytes, char* err, size_t cap) {
    if (!element_bytes(dtype)) return fail(PV_EARG, err, cap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (B < 0 || T < 1 || D < 0) return fail(PV_EARG, err, cap, "shape: B >= 0, T >= 1, D >= 0");
    if (B > 65535 || chunks_of(T) > 65535 || D > int64_t(BLOCK) * INT32_MAX) return fail(PV_EARG, err, cap, "shape: too large");
    if (B && D && (!work || work_bytes < pv_gated_scan_work_bytes(B, T, D))) return fail(PV_EARG, err, cap, "work: too small");
    return PV_OK;
}

}  // namespace

extern "C" {

int64_t pv_gated_scan_chunks(int64_t T) { return T > 0 ? chunks_of(T) : 0; }
uint64_t pv_gated_scan_work_bytes(int64_t B, int64_t T, int64_t D) {
    return B > 0 && T > 0 && D > 0 ? uint64_t(B) * uint64_t(chunks_of(T)) * uint64_t(D) * 12 : 0;
}

int32_t pv_gated_scan_hip(const void* gate, const void* value, const float* state, const uint8_t* reset, int64_t B, int64_t T, int64_t D, int64_t gate_b,
                          int64_t gate_t, int64_t value_b, int64_t value_t, int32_t dtype, void* out, float* last, float* carry, void* work,
                          uint64_t work_bytes, void* stream, char* err, size_t errcap) {
    if (int32_t e = check(B, T, D, dtype, work, work_bytes, err, errcap)) return e;
    if (!B || !D) return PV_OK;
    if (!gate || !value || !out || !last) return fail(PV_EARG, err, errcap, "null argument");
    const Shape S{B, T, D, gate_b, gate_t, value_b, value_t, 0, 0, chunks_of(T)};
    const hipStream_t st = hipStream_t(stream);
    float2* maps = static_cast<float2*>(work);
    if (!carry) carry = reinterpret_cast<float*>(maps + B * S.chunks * D);
    const dim3 grid((D + BLOCK - 1) / BLOCK, S.chunks, B), rows(grid.x, B);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        scan_map_kernel<E><<<grid, BLOCK, 0, st>>>(S, static_cast<const E*>(gate), static_cast<const E*>(value), reset, maps);
        scan_carry_kernel<<<rows, BLOCK, 0, st>>>(S, maps, state, carry);
        scan_apply_kernel<E><<<grid, BLOCK, 0, st>>>(S, static_cast<const E*>(gate), static_cast<const E*>(value), reset, carry, static_cast<E*>(out), last);
        return launched(err, errcap);
    });
}

int32_t pv_gated_scan_backward_hip(const void* gate, const void* value, const float* carry, const uint8_t* reset, int64_t B, int64_t T, int64_t D,
                                   int64_t gate_b, int64_t gate_t, int64_t value_b, int64_t value_t, const void* d_out, int64_t d_out_b, int64_t d_out_t,
                                   const float* d_last, int32_t dtype, void* d_gate, void* d_value, float* d_state, void* work, uint64_t work_bytes,
                                   void* stream, char* err, size_t errcap) {
    if (int32_t e = check(B, T, D, dtype, work, work_bytes, err, errcap)) return e;
    if (!B || !D) return PV_OK;
    if (!gate || !value || !carry || !d_out || !d_gate || !d_value) return fail(PV_EARG, err, errcap, "null argument");
    const Shape S{B, T, D, gate_b, gate_t, value_b, value_t, d_out_b, d_out_t, chunks_of(T)};
    const hipStream_t st = hipStream_t(stream);
    float2* maps = static_cast<float2*>(work);
    float* flow = reinterpret_cast<float*>(maps + B * S.chunks * D);
    const dim3 grid((D + BLOCK - 1) / BLOCK, S.chunks, B), rows(grid.x, B);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        scan_back_map_kernel<E><<<grid, BLOCK, 0, st>>>(S, static_cast<const E*>(gate), static_cast<const E*>(d_out), reset, maps);
        scan_back_carry_kernel<<<rows, BLOCK, 0, st>>>(S, maps, d_last, flow);
        scan_back_apply_kernel<E><<<grid, BLOCK, 0, st>>>(S, static_cast<const E*>(gate), static_cast<const E*>(value), reset, carry, flow,
                                                          static_cast<const E*>(d_out), static_cast<E*>(d_gate), static_cast<E*>(d_value), d_state);
        return launched(err, errcap);
    });
}

}  // extern "C"
