// Dropout from the counter stream of draws.hip, forward and backward, with the mask never stored.
//
// Element e = first + i of the global tensor takes 32 bits of the 64-bit word mix(key + (e >> 1) * GAMMA) -- the low half
// for an even e, the high half for an odd one; mix is the splitmix64 finaliser counter_uniform uses -- and is kept iff
// those bits are >= round(p 2^32).  So the mask is a function of (key, global element) alone: the backward pass, a replay
// and any sharding of the batch see the same one, and a second evaluation costs less than a byte per element would.
//   y = keep ? x / (1 - p) : 0        (+ residual)
// A dropped element is 0 whatever x holds there (an infinity or NaN in a dropped place does not pass).
//
// Bound by HBM: 786432 x 256 bf16 in 130 us, 6.2 TB/s; 16383 x 2047 bf16 with a residual in 31 us, 6.4 TB/s.  The generator
// is not far behind: two elements take six quarter-rate multiplications (24 x 16 of about 700 cycles a piece of 8), 110 us
// of this case if nothing else did anything.  As 64-bit arithmetic with a 64-bit comparison the kernel took 162 us; as a
// grid that strides over the array, 187.
#include <math.h>

#include "rows.h"

namespace {

using nerf::Row;

constexpr uint64_t GAMMA = 0xD1342543DE82EF95ull;

// The finaliser on 32-bit halves: its 64-bit shifts as an align and a shift, which run at full rate.
struct Word {
    uint32_t lo, hi;
};

template <int SHIFT>
__device__ __forceinline__ Word fold(Word x) {               // x ^ (x >> SHIFT)
    return {x.lo ^ __builtin_amdgcn_alignbit(x.hi, x.lo, SHIFT), x.hi ^ (x.hi >> SHIFT)};
}

__device__ __forceinline__ Word times(Word x, uint64_t c) {
    const uint64_t low = (uint64_t)x.lo * (uint32_t)c;
    return {(uint32_t)low, (uint32_t)(low >> 32) + x.lo * (uint32_t)(c >> 32) + x.hi * (uint32_t)c};
}

__device__ __forceinline__ Word mix(uint64_t state) {
    Word x = {(uint32_t)state, (uint32_t)(state >> 32)};
    x = times(fold<30>(x), 0xBF58476D1CE4E5B9ull);
    x = times(fold<27>(x), 0x94D049BB133111EBull);
    return fold<31>(x);
}

// A piece a thread.  ODD: the global index of element 0 is odd, so that every pair of elements takes halves of two words.
template <typename T, bool ODD, bool ADD>
__global__ __launch_bounds__(256) void dropout_kernel(const T *__restrict__ x, const T *__restrict__ residual, int64_t n,
                                                      uint32_t threshold, bool none, float scale, uint64_t key,
                                                      const uint64_t *__restrict__ key_dev, int64_t first,
                                                      T *__restrict__ out) {
    constexpr int VEC = Row<T>::VEC, WORDS = VEC / 2 + (ODD ? 1 : 0);
    if (key_dev) key = *key_dev;
    const int64_t pieces = n / VEC, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < pieces) {
        const int64_t at = i * VEC;
        const Row<T> a = nerf::load_16<T>(x + at);
        Row<T> r;
        if (ADD) r = nerf::load_16<T>(residual + at);
        // (first + at) / 2 in a part that is the workgroup's and one that is the thread's: a multiplication less a thread
        uint64_t state = key + ((uint64_t)(first >> 1) + (uint64_t)blockIdx.x * (256 * VEC / 2)) * GAMMA +
                         (uint64_t)(threadIdx.x * (VEC / 2)) * GAMMA;
        uint32_t bits[2 * WORDS];
#pragma unroll
        for (int j = 0; j < WORDS; ++j) {
            const Word w = mix(state);
            bits[2 * j] = w.lo;
            bits[2 * j + 1] = w.hi;
            state += GAMMA;
        }
        Row<T> y;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float v = bits[j + (ODD ? 1 : 0)] >= threshold && !none ? (float)a.v[j] * scale : 0.0f;
            y.v[j] = (T)(ADD ? (float)r.v[j] + v : v);
        }
        nerf::store_16(out + at, y);
    }
    // what is left behind the last whole piece
    const int64_t at = pieces * VEC + threadIdx.x;
    if (blockIdx.x == 0 && at < n) {
        const Word w = mix(key + (uint64_t)((first + at) >> 1) * GAMMA);
        const float v = (((first + at) & 1) ? w.hi : w.lo) >= threshold && !none ? (float)x[at] * scale : 0.0f;
        out[at] = (T)(ADD ? (float)residual[at] + v : v);
    }
}

template <typename T>
void launch(const void *x, const void *residual, int64_t n, uint32_t threshold, bool none, float scale, uint64_t key,
            const uint64_t *key_dev, int64_t first, void *out, hipStream_t stream) {
    auto kernel = residual ? ((first & 1) ? dropout_kernel<T, true, true> : dropout_kernel<T, false, true>)
                           : ((first & 1) ? dropout_kernel<T, true, false> : dropout_kernel<T, false, false>);
    constexpr int64_t MOST = (int64_t)1 << 31;               // of one launch, whose threads are counted in 32 bits
    for (int64_t at = 0; at < n; at += MOST) {
        const int64_t count = n - at < MOST ? n - at : MOST, pieces = (count + Row<T>::VEC - 1) / Row<T>::VEC;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, stream, static_cast<const T *>(x) + at,
                           residual ? static_cast<const T *>(residual) + at : nullptr, count, threshold, none, scale, key, key_dev,
                           first + at, static_cast<T *>(out) + at);
    }
}

}  // namespace

NERF_API int nerf_dropout(const void *x, const void *residual, int dtype, int64_t n, double p, uint64_t key,
                          const uint64_t *key_dev, int64_t first, void *out, nerf_stream_t stream) {
    NERF_REQUIRE(nerf::known_dtype(dtype), "nerf_dropout: unknown dtype");
    NERF_REQUIRE(n >= 0 && n <= (int64_t)1 << 40 && first >= 0 && first <= INT64_MAX - n, "nerf_dropout: element range out of bounds");
    NERF_REQUIRE(p >= 0.0 && p <= 1.0, "nerf_dropout: p must be in [0, 1]");
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(x && out, "nerf_dropout: null pointer");
    const uint64_t threshold = (uint64_t)floor(p * 4294967296.0 + 0.5);      // 2^32 (p = 1): nothing is kept
    const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    NERF_FOR_DTYPE(dtype, T, launch<T>(x, residual, n, (uint32_t)threshold, threshold >> 32, scale, key, key_dev, first, out,
                                       nerf::as_stream(stream)));
    return nerf::check_launch("nerf_dropout");
}
