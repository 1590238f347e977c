// Rows of fp32 / bf16 / fp16 values for the learned-code operators (layernorm.hip, dropout.hip, embedding.hip).
//
// A row is moved in 16-byte pieces per lane whatever its address: gfx950 serves a global dwordx4 access at any element
// boundary, so an odd row length needs no variant of its own.  Only the piece that a row ends in goes value by value:
// nothing is read or written beyond a row.  Arithmetic is fp32; a value is rounded once, when it is stored.
#pragma once
#include "common.h"

namespace nerf {

template <typename T>
struct Row {
    static constexpr int VEC = 16 / (int)sizeof(T);
    T v[VEC];
};

// `count` values (any number; <= 0: none) starting at p; missing ones read as 0
template <typename T>
__device__ __forceinline__ Row<T> load_piece(const T *p, int64_t count) {
    Row<T> r;
    if (count >= Row<T>::VEC) {
        __builtin_memcpy(&r, p, 16);
    } else {
#pragma unroll
        for (int j = 0; j < Row<T>::VEC; ++j) r.v[j] = j < count ? p[j] : (T)0.0f;
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void store_piece(T *p, const Row<T> &r, int64_t count) {
    if (count >= Row<T>::VEC) {
        __builtin_memcpy(p, &r, 16);
    } else {
#pragma unroll
        for (int j = 0; j < Row<T>::VEC; ++j)
            if (j < count) p[j] = r.v[j];
    }
}

// VEC consecutive weights as fp32: of the row's own type, or fp32
template <typename T>
__device__ __forceinline__ void load_weights(const void *w, bool w_f32, int64_t at, int64_t count, float absent,
                                             float (&out)[Row<T>::VEC]) {
    constexpr int VEC = Row<T>::VEC;
    if (w == nullptr) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = absent;
    } else if (sizeof(T) == 2 && w_f32) {
        const float *p = static_cast<const float *>(w) + at;
#pragma unroll
        for (int h = 0; h < VEC; h += 4) {
            const Row<float> r = load_piece(p + h, count - h);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[h + j] = r.v[j];
        }
    } else {
        const Row<T> r = load_piece(static_cast<const T *>(w) + at, count);
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = (float)r.v[j];
    }
}

// sum over groups of WIDTH lanes (a power of two <= 64), every lane gets it
template <int WIDTH>
__device__ __forceinline__ float lane_sum(float x) {
#pragma unroll
    for (int d = 1; d < WIDTH; d <<= 1) x += __shfl_xor(x, d, WAVE);
    return x;
}

inline bool known_dtype(int t) { return t == NERF_F32 || t == NERF_BF16 || t == NERF_F16; }
inline int dtype_bytes(int t) { return t == NERF_F32 ? 4 : 2; }

}  // namespace nerf

// call f<T>(...) for the element type of a NERF_* code that known_dtype() accepted
#define NERF_FOR_DTYPE(code, T, ...)                        \
    do {                                                    \
        if ((code) == NERF_F32) { using T = float; __VA_ARGS__; }   \
        else if ((code) == NERF_BF16) { using T = __bf16; __VA_ARGS__; } \
        else { using T = _Float16; __VA_ARGS__; }           \
    } while (0)
