// Dropout without a stored mask: an element's 16 bits are a function of a seed, a site and the element's index alone, so that the
// backward pass, another cut into lanes or another operator makes the same ones again.
//
// The bits are those of the counter-based generator of four 32-bit words in ten rounds by Salmon, Moraes, Dror and Shaw
// ("Parallel random numbers: as easy as 1, 2, 3", SC 2011), of key `seed` and counter (index / 8 in 64 bits, site, 0): eight
// elements to a counter, a word's low half first. An element is dropped where its bits are below `least` = round(p 2^16), else
// multiplied by 2^16 / (2^16 - least), 1 over the share that is kept. (16 bits an element: a wave makes those of 512 elements in
// some 450 cycles, 20 products of 32 x 32 bits at a quarter of the rate; 32 bits an element would take as long as the bytes.)
#pragma once
#include "pv_ops.h"

namespace pvo {

struct Drop {
    const uint64_t* at;                    // the seed in memory, or null: `value`
    uint64_t value;
    uint32_t site, least;
    float up;
    __device__ uint64_t seed() const { return at ? *at : value; }
};

inline Drop drop_of(const int64_t* at, int64_t value, uint32_t site, double p) {
    const uint32_t least = uint32_t(p * 65536.0 + 0.5);
    return {reinterpret_cast<const uint64_t*>(at), uint64_t(value), site, least, least < 65536 ? float(65536.0 / (65536 - least)) : 0.0f};
}

// The 16 bits of elements 8 block .. 8 block + 7, two to a word
struct Bits { uint32_t w[4]; };
__device__ inline Bits bits_of(uint64_t seed, uint64_t block, uint32_t site) {
    uint32_t a = uint32_t(block), b = uint32_t(block >> 32), c = site, d = 0, k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; round++) {
        const uint64_t x = uint64_t(a) * 0xD2511F53u, y = uint64_t(c) * 0xCD9E8D57u;
        a = uint32_t(y >> 32) ^ b ^ k0;
        b = uint32_t(y);
        c = uint32_t(x >> 32) ^ d ^ k1;
        d = uint32_t(x);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{a, b, c, d}};
}

// f(j, kept) for the P elements from index `first` on (P at most 8): of one counter, or of two where they begin inside one
template <int P, typename F> __device__ inline void each_kept(const Drop& drop, uint64_t seed, uint64_t first, F&& f) {
    static_assert(P <= 8, "two counters at most");
    const uint32_t off = uint32_t(first) & 7;
    const Bits lo = bits_of(seed, first >> 3, drop.site);
    if (off + P <= 8) {
        if constexpr (P == 8) {
#pragma unroll
            for (int j = 0; j < 8; j++) f(j, (j & 1 ? lo.w[j / 2] >> 16 : lo.w[j / 2] & 0xffff) >= drop.least);
            return;
        }
    }
    Bits hi = lo;
    if (off + P > 8) hi = bits_of(seed, (first >> 3) + 1, drop.site);
#pragma unroll
    for (int j = 0; j < P; j++) {          // (words chosen by compares: an index that is not known would put them into memory)
        const uint32_t e = off + j, k = e / 2;
        uint32_t w = lo.w[0];
        w = k == 1 ? lo.w[1] : w;
        w = k == 2 ? lo.w[2] : w;
        w = k == 3 ? lo.w[3] : w;
        w = k == 4 ? hi.w[0] : w;
        w = k == 5 ? hi.w[1] : w;
        w = k == 6 ? hi.w[2] : w;
        w = k == 7 ? hi.w[3] : w;
        f(j, (e & 1 ? w >> 16 : w & 0xffff) >= drop.least);
    }
}

// What is wrong with a call's p, or null
inline const char* drop_error(double p) { return p >= 0.0 && p <= 1.0 ? nullptr : "p: 0 <= p <= 1"; }

}  // namespace pvo
