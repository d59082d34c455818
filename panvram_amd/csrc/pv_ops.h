// What the operators' kernels (pv_scan.hip, pv_norm.hip, pv_loss.hip, pv_clip.hip) share: element types, wide loads and
// stores, wave sums, and the checks of a C entry.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include "../../include/panvram_amd.h"

namespace pvo {

constexpr int WAVE = 64;

// What the kernels hold one element as: PV_F32, PV_BF16, PV_F16. Conversions from float round to nearest even.
using bf16 = __bf16;
using f16 = _Float16;

template <int BYTES> struct raw_of;
template <> struct raw_of<1> { using type = uint8_t; };
template <> struct raw_of<2> { using type = uint16_t; };
template <> struct raw_of<4> { using type = uint32_t; };
template <> struct raw_of<8> { using type = __attribute__((ext_vector_type(2))) uint32_t; };
template <> struct raw_of<16> { using type = __attribute__((ext_vector_type(4))) uint32_t; };
template <> struct raw_of<32> { using type = __attribute__((ext_vector_type(8))) uint32_t; };      // (two loads)

// N elements moved by one load or store of N * sizeof(T) bytes, from any address that an element may have: the compiler knows that
// gfx950 takes global accesses off their own size's alignment, and makes one of each
template <typename T, int N> struct pack {
    using raw = typename raw_of<int(sizeof(T)) * N>::type;
    struct __attribute__((packed, aligned(sizeof(T)))) at_element { raw bits; };
    union { raw bits; T v[N]; };
    __device__ static pack load(const T* p) { pack r; r.bits = reinterpret_cast<const at_element*>(p)->bits; return r; }
    __device__ void store(T* p) const { reinterpret_cast<at_element*>(p)->bits = bits; }
    // the same past the caches, for what is not used again soon
    __device__ static pack load_once(const T* p) { pack r; r.bits = __builtin_nontemporal_load(&reinterpret_cast<const at_element*>(p)->bits); return r; }
    __device__ void store_once(T* p) const { __builtin_nontemporal_store(bits, &reinterpret_cast<at_element*>(p)->bits); }
    // the same of the first `left` elements, where there are fewer than N: one by one, the others 0 and not written
    __device__ static pack load_part(const T* p, int64_t left) {
        pack r;
#pragma unroll
        for (int j = 0; j < N; j++) r.v[j] = j < left ? p[j] : T(0.0f);
        return r;
    }
    __device__ void store_part(T* p, int64_t left) const {
#pragma unroll
        for (int j = 0; j < N; j++) if (j < left) p[j] = v[j];
    }
};

inline bool aligned(const void* p, uint64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

__device__ inline float wave_sum(float x) {
#pragma unroll
    for (int d = WAVE / 2; d; d >>= 1) x += __shfl_xor(x, d, WAVE);
    return x;
}

// A launch's work items: HIP takes fewer than 2^32
constexpr int64_t MOST_ITEMS = int64_t(1) << 32;

inline int32_t fail(int32_t code, char* err, size_t cap, const char* m) {
    if (err && cap) snprintf(err, cap, "%s", m);
    return code;
}

// The last launch's error as a status code
inline int32_t launched(char* err, size_t cap) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? PV_OK : fail(PV_EHIP, err, cap, hipGetErrorString(e));
}

inline int element_bytes(int32_t dtype) { return dtype == PV_F32 ? 4 : dtype == PV_BF16 || dtype == PV_F16 ? 2 : 0; }

// f.template operator()<T>() of the element type `dtype` names (checked before)
template <typename F> int32_t with_type(int32_t dtype, F&& f) {
    if (dtype == PV_F32) return f(float{});
    if (dtype == PV_BF16) return f(bf16{});
    return f(f16{});
}

}  // namespace pvo
