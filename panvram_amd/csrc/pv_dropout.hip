// Dropout of a tensor by a counter-based generator (pv_drop.h): y[i] = kept(i) ? x[i] / (1 - p) : 0. The gradient is the same of d_y.
//
// Each lane has the eight elements of one counter: it makes their bits, reads 16 bytes (32 in float32) and writes as many, past the
// caches. What bounds it: the bytes, with the generator's products beside them. 65,536 x 1,024 bfloat16: 42 us, 6.4 TB/s.
#include "pv_drop.h"

#include <algorithm>

using namespace pvo;

namespace {

constexpr int BLOCK = 256;

template <typename E>
__global__ __launch_bounds__(BLOCK) void dropout_kernel(const E* __restrict__ x, int64_t n, uint64_t block0, Drop drop, E* __restrict__ y) {
    const int64_t i = (int64_t(blockIdx.x) * BLOCK + threadIdx.x) * 8;
    if (i >= n) return;
    const bool whole = i + 8 <= n;
    pack<E, 8> v = whole ? pack<E, 8>::load_once(x + i) : pack<E, 8>::load_part(x + i, n - i);
    each_kept<8>(drop, drop.seed(), (block0 << 3) + uint64_t(i), [&](int j, bool kept) { v.v[j] = kept ? E(float(v.v[j]) * drop.up) : E(0.0f); });
    if (whole) v.store_once(y + i);
    else v.store_part(y + i, n - i);
}

}  // namespace

extern "C" int32_t pv_dropout_hip(const void* x, int64_t n, double p, const int64_t* seed_at, int64_t seed, uint32_t site, int32_t dtype, void* y, void* stream,
                                  char* err, size_t errcap) {
    const int bytes = element_bytes(dtype);
    if (!bytes) return fail(PV_EARG, err, errcap, "dtype: one of PV_F32, PV_BF16, PV_F16");
    if (n < 0 || n > int64_t(1) << 48) return fail(PV_EARG, err, errcap, "shape: 0 <= n <= 2^48");
    if (const char* m = drop_error(p)) return fail(PV_EARG, err, errcap, m);
    if (!n) return PV_OK;
    if (!x || !y) return fail(PV_EARG, err, errcap, "null argument");
    if (!aligned(x, bytes) || !aligned(y, bytes) || !aligned(seed_at, 8)) return fail(PV_EARG, err, errcap, "address: not a multiple of the element's size");
    const Drop drop = drop_of(seed_at, seed, site, p);
    return with_type(dtype, [&](auto e) {
        using E = decltype(e);
        constexpr int64_t MOST = (MOST_ITEMS - BLOCK) * 8;                     // elements of a launch, whole counters
        for (int64_t i = 0; i < n; i += MOST) {
            const int64_t part = std::min(n - i, MOST), lanes = (part + 7) / 8;
            dropout_kernel<E><<<dim3((lanes + BLOCK - 1) / BLOCK), BLOCK, 0, hipStream_t(stream)>>>(static_cast<const E*>(x) + i, part, uint64_t(i) / 8, drop,
                                                                                                   static_cast<E*>(y) + i);
        }
        return launched(err, errcap);
    });
}
