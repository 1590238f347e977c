// Dropout from the counter stream of draws.hip, forward and backward, with the mask never stored.
//
// Element e = first + i of the global tensor takes 32 bits of the 64-bit word mix(key + (e >> 1) * GAMMA) -- the low half
// for an even e, the high half for an odd one; mix is the splitmix64 finaliser counter_uniform uses -- and is kept iff
// those bits are >= round(p 2^32).  So the mask is a function of (key, global element) alone: the backward pass, a replay
// and any sharding of the batch see the same one, and a second evaluation costs less than a byte per element would.
//   y = keep ? x / (1 - p) : 0        (+ residual)
// A dropped element is 0 whatever x holds there (an infinity or NaN in a dropped place does not pass).
#include <math.h>

#include "rows.h"

namespace {

using nerf::Row;

constexpr uint64_t GAMMA = 0xD1342543DE82EF95ull;

__device__ __forceinline__ uint64_t mix(uint64_t x) {
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    return x ^ (x >> 31);
}

// ODD: the global index of element 0 is odd, so that every pair of elements takes halves of two words
template <typename T, bool ODD, bool ADD>
__global__ __launch_bounds__(256) void dropout_kernel(const T *__restrict__ x, const T *__restrict__ residual, int64_t n,
                                                      uint64_t threshold, float scale, uint64_t key,
                                                      const uint64_t *__restrict__ key_dev, int64_t first,
                                                      T *__restrict__ out) {
    constexpr int VEC = Row<T>::VEC, WORDS = VEC / 2 + (ODD ? 1 : 0);
    if (key_dev) key = *key_dev;
    const int64_t pieces = (n + VEC - 1) / VEC;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t at = i * VEC, count = n - at;
        const Row<T> a = nerf::load_flat(x + at, count);
        Row<T> r;
        if (ADD) r = nerf::load_flat(residual + at, count);
        uint64_t state = key + (uint64_t)((first + at) >> 1) * GAMMA;
        uint32_t bits[2 * WORDS];
#pragma unroll
        for (int j = 0; j < WORDS; ++j) {
            const uint64_t w = mix(state);
            bits[2 * j] = (uint32_t)w;
            bits[2 * j + 1] = (uint32_t)(w >> 32);
            state += GAMMA;
        }
        Row<T> y;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const bool keep = bits[j + (ODD ? 1 : 0)] >= threshold;
            const float v = keep ? (float)a.v[j] * scale : 0.0f;
            y.v[j] = (T)(ADD ? (float)r.v[j] + v : v);
        }
        nerf::store_flat(out + at, y, count);
    }
}

template <typename T>
void launch(const void *x, const void *residual, int64_t n, uint64_t threshold, float scale, uint64_t key,
            const uint64_t *key_dev, int64_t first, void *out, hipStream_t stream) {
    const int64_t pieces = (n + Row<T>::VEC - 1) / Row<T>::VEC;
    int64_t grid = (pieces + 255) / 256;
    if (grid > 256 * 16) grid = 256 * 16;
    auto kernel = residual ? ((first & 1) ? dropout_kernel<T, true, true> : dropout_kernel<T, false, true>)
                           : ((first & 1) ? dropout_kernel<T, true, false> : dropout_kernel<T, false, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, stream, static_cast<const T *>(x),
                       static_cast<const T *>(residual), n, threshold, scale, key, key_dev, first, static_cast<T *>(out));
}

}  // namespace

NERF_API int nerf_dropout(const void *x, const void *residual, int dtype, int64_t n, double p, uint64_t key,
                          const uint64_t *key_dev, int64_t first, void *out, nerf_stream_t stream) {
    NERF_REQUIRE(nerf::known_dtype(dtype), "nerf_dropout: unknown dtype");
    NERF_REQUIRE(n >= 0 && first >= 0 && first <= INT64_MAX - n, "nerf_dropout: element range out of bounds");
    NERF_REQUIRE(p >= 0.0 && p <= 1.0, "nerf_dropout: p must be in [0, 1]");
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(x && out, "nerf_dropout: null pointer");
    const uint64_t threshold = (uint64_t)floor(p * 4294967296.0 + 0.5);      // 2^32 (p = 1): nothing is kept
    const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    NERF_FOR_DTYPE(dtype, T, launch<T>(x, residual, n, threshold, scale, key, key_dev, first, out, nerf::as_stream(stream)));
    return nerf::check_launch("nerf_dropout");
}
