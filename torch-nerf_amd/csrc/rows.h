// Rows of fp32 / bf16 / fp16 values for the learned-code operators (layernorm.hip, dropout.hip, embedding.hip).
//
// A row is moved in 16-byte pieces per lane whatever its address: gfx950 serves a global dwordx4 access at any element
// boundary, so an odd row length needs no variant of its own.  The piece that a row ends in is moved back to end with the
// row: it holds some values of its neighbour again (`Place::own` tells them apart), so that no access goes value by value
// and none leaves the row.  Only rows shorter than a piece (TINY) do.  Arithmetic is fp32; a value is rounded once, when
// it is stored.
#pragma once
#include "common.h"

namespace nerf {

template <typename T>
struct Row {
    static constexpr int VEC = 16 / (int)sizeof(T);
    T v[VEC];
};

// One 16-byte access at an element's alignment.  As a vector of words: a copy value by value is taken apart by the compiler
// where only some values are used on some path.
typedef uint32_t words __attribute__((ext_vector_type(4)));
typedef words loose_words __attribute__((aligned(2)));

template <typename T>
__device__ __forceinline__ Row<T> load_16(const void *p) {
    return __builtin_bit_cast(Row<T>, static_cast<words>(*static_cast<const loose_words *>(p)));
}

template <typename T>
__device__ __forceinline__ void store_16(void *p, const Row<T> &r) {
    *static_cast<loose_words *>(p) = __builtin_bit_cast(words, r);
}

// Where the piece that would begin at value `a` of a row of C values is: at `at`, with its first `skip` values another's.
// skip >= VEC: the row ends before it.
template <typename T, bool TINY>
struct Place {
    int at, skip, C;
    __device__ __forceinline__ Place(int a, int C_) : at(TINY ? a : (a < C_ - Row<T>::VEC ? a : C_ - Row<T>::VEC)), skip(a - at), C(C_) {}
    __device__ __forceinline__ bool live() const { return TINY ? at < C : skip < Row<T>::VEC; }
    // unsigned: a uniform row pointer then stays in scalar registers, with 32 bits per lane beside it
    __device__ __forceinline__ uint32_t bytes() const { return (uint32_t)at * (uint32_t)sizeof(T); }
    __device__ __forceinline__ bool own(int j) const { return TINY ? at + j < C : j >= skip; }
};

template <bool TINY, typename T>
__device__ __forceinline__ Row<T> load_piece(const T *row, const Place<T, TINY> &p) {
    Row<T> r;
    if (TINY) {
#pragma unroll
        for (int j = 0; j < Row<T>::VEC; ++j) r.v[j] = p.own(j) ? row[p.at + j] : (T)0.0f;
    } else {
        r = load_16<T>(reinterpret_cast<const char *>(row) + p.bytes());
    }
    return r;
}

// (values shared with the neighbouring piece are stored twice, the same)
template <bool TINY, typename T>
__device__ __forceinline__ void store_piece(T *row, const Place<T, TINY> &p, const Row<T> &r) {
    if (TINY) {
#pragma unroll
        for (int j = 0; j < Row<T>::VEC; ++j)
            if (p.own(j)) row[p.at + j] = r.v[j];
    } else if (p.live()) {
        store_16(reinterpret_cast<char *>(row) + p.bytes(), r);
    }
}

// the same piece of the weights, as fp32: of the row's own type, or fp32; `absent` where there are none
template <bool TINY, typename T>
__device__ __forceinline__ void load_weights(const void *w, bool w_f32, const Place<T, TINY> &p, float absent,
                                             float (&out)[Row<T>::VEC]) {
    constexpr int VEC = Row<T>::VEC;
    if (w == nullptr) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = absent;
    } else if (sizeof(T) == 2 && w_f32) {
        const float *f = reinterpret_cast<const float *>(static_cast<const char *>(w) + (uint32_t)p.at * 4u);
        if (TINY) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) out[j] = p.own(j) ? f[j] : 0.0f;
        } else {
            __builtin_memcpy(out, f, VEC * 4);
        }
    } else {
        const Row<T> r = load_piece<TINY>(static_cast<const T *>(w), p);
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = (float)r.v[j];
    }
}

// Sum over groups of WIDTH lanes (a power of two <= 64), every lane gets it.  In the vector ALU alone: inside of 16 lanes by
// DPP (quad permutes, then mirrors: the quads agree by then, so a mirror is as good as an exchange), across them by gfx950's
// row and half swaps.  Six steps of ds_bpermute take ten times as long, and a row's sums are in every row's way.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

template <int WIDTH>
__device__ __forceinline__ float lane_sum(float x) {
    if constexpr (WIDTH >= 2) x = dpp_add<0xB1>(x);          // quad_perm [1, 0, 3, 2]
    if constexpr (WIDTH >= 4) x = dpp_add<0x4E>(x);          // quad_perm [2, 3, 0, 1]
    if constexpr (WIDTH >= 8) x = dpp_add<0x141>(x);         // row_half_mirror
    if constexpr (WIDTH >= 16) x = dpp_add<0x140>(x);        // row_mirror
    if constexpr (WIDTH >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);     // {rows 0 0 2 2, rows 1 1 3 3}
        x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    }
    if constexpr (WIDTH >= 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);     // {low half twice, high half twice}
        x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
    }
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
