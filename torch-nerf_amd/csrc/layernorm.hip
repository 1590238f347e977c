// Layer norm over the last axis, forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   y = (x - mu) r w + b,   mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps)
//   gx = r (q - mean(q) - h mean(q h)),  q = g w, h = (x - mu) r;   gw = sum_rows g h,   gb = sum_rows g
//
// A row stays in registers between its one read and its one write: TPR lanes hold it as NV 16-byte pieces each.  The
// variance is taken about the mean (a second sum over the registers), so a large offset costs no digits.  Statistics and
// sums are fp32.  Rows of up to 64 lanes need no barrier; a longer row takes a workgroup.
#include "rows.h"

#ifndef X_AHEAD
#define X_AHEAD 0
#endif
namespace {

using nerf::Row;

// Sum of K values over the TPR lanes that share a row.  TPR > 64: through LDS, every group of TPR threads of the workgroup
// at once; `slot` alternates so that one barrier per sum is enough (a wave that runs ahead writes the other half of `red`).
template <int TPR, int K, int BLOCK>
__device__ __forceinline__ void row_sum(float (&v)[K], float *red, int &slot) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = nerf::lane_sum<(TPR < WAVE ? TPR : WAVE)>(v[k]);
    if constexpr (TPR > WAVE) {
        constexpr int WAVES = TPR / WAVE;
        float *r = red + slot * (BLOCK / WAVE) * K;
        slot ^= 1;
        if ((threadIdx.x & (WAVE - 1)) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) r[(threadIdx.x / WAVE) * K + k] = v[k];
        }
        __syncthreads();
        r += threadIdx.x / TPR * WAVES * K;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) s += r[w * K + k];
            v[k] = s;
        }
    }
}

// The compiler may not keep what it made of p (or loaded through p) before this point.
template <typename T>
__device__ __forceinline__ void forget(Row<T> &p) {
    uint32_t u[4];
    __builtin_memcpy(u, &p, 16);
    asm volatile("" : "+v"(u[0]), "+v"(u[1]), "+v"(u[2]), "+v"(u[3]));
    __builtin_memcpy(&p, u, 16);
}

template <typename T, int TPR, int NV, int BLOCK, bool TINY>
__global__ __launch_bounds__(BLOCK) void layernorm_kernel(const T *__restrict__ x, int64_t x_stride, int64_t M, int C,
                                                          const void *__restrict__ weight, const void *__restrict__ bias,
                                                          int w_f32, float eps, T *__restrict__ y,
                                                          float *__restrict__ mean, float *__restrict__ rstd) {
    constexpr int VEC = Row<T>::VEC, RPB = BLOCK / TPR;
    constexpr bool HOIST = NV * VEC <= 8;                     // the weights stay in registers from row to row
    static_assert(TPR <= WAVE || TPR == BLOCK, "a row beyond one wavefront takes the whole workgroup");
    __shared__ float red[TPR > WAVE ? 2 * (BLOCK / WAVE) : 1];
    int slot = 0;
    const int lane = threadIdx.x % TPR;
    const float inv_c = 1.0f / (float)C;
    float w[HOIST ? NV : 1][VEC], b[HOIST ? NV : 1][VEC];
    if constexpr (HOIST) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * TPR + lane) * VEC, C);
            nerf::load_weights<TINY, T>(weight, w_f32, at, 1.0f, w[i]);
            nerf::load_weights<TINY, T>(bias, w_f32, at, 0.0f, b[i]);
        }
    }
    for (int64_t row = (int64_t)blockIdx.x * RPB + nerf::lane_group<TPR>(); row < M; row += (int64_t)gridDim.x * RPB) {
        float v[NV][VEC], s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * TPR + lane) * VEC, C);
            const Row<T> p = nerf::load_piece<TINY>(x + row * x_stride, at);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i][j] = (float)p.v[j];
                s[0] += at.own(j) ? v[i][j] : 0.0f;
            }
        }
        row_sum<TPR, 1, BLOCK>(s, red, slot);
        const float mu = s[0] * inv_c;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * TPR + lane) * VEC, C);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i][j] -= mu;
                const float d = at.own(j) ? v[i][j] : 0.0f;
                s[0] = fmaf(d, d, s[0]);
            }
        }
        row_sum<TPR, 1, BLOCK>(s, red, slot);
        const float r = 1.0f / sqrtf(s[0] * inv_c + eps);
        if (lane == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * TPR + lane) * VEC, C);
            if constexpr (!HOIST) {
                nerf::load_weights<TINY, T>(weight, w_f32, at, 1.0f, w[0]);
                nerf::load_weights<TINY, T>(bias, w_f32, at, 0.0f, b[0]);
            }
            Row<T> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.v[j] = (T)fmaf(v[i][j] * r, w[HOIST ? i : 0][j], b[HOIST ? i : 0][j]);
            nerf::store_piece<TINY>(y + row * C, at, o);
        }
    }
}

// Rows longer than a workgroup's registers: three sweeps over the row (the second and third from cache).
template <typename T>
__global__ __launch_bounds__(1024) void layernorm_long_kernel(const T *__restrict__ x, int64_t x_stride, int64_t M, int C,
                                                              const void *__restrict__ weight,
                                                              const void *__restrict__ bias, int w_f32, float eps,
                                                              T *__restrict__ y, float *__restrict__ mean,
                                                              float *__restrict__ rstd) {
    constexpr int VEC = Row<T>::VEC;
    __shared__ float red[2 * 16];
    int slot = 0;
    const float inv_c = (float)(1.0 / (double)C);
    for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
        const T *xr = x + row * x_stride;
        float s[1] = {0.0f};
        for (int a = threadIdx.x * VEC; a < C; a += 1024 * VEC) {
            const nerf::Place<T, false> at(a, C);
            const Row<T> p = nerf::load_piece<false>(xr, at);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[0] += at.own(j) ? (float)p.v[j] : 0.0f;
        }
        row_sum<1024, 1, 1024>(s, red, slot);
        const float mu = s[0] * inv_c;
        s[0] = 0.0f;
        for (int a = threadIdx.x * VEC; a < C; a += 1024 * VEC) {
            const nerf::Place<T, false> at(a, C);
            const Row<T> p = nerf::load_piece<false>(xr, at);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = at.own(j) ? (float)p.v[j] - mu : 0.0f;
                s[0] = fmaf(d, d, s[0]);
            }
        }
        row_sum<1024, 1, 1024>(s, red, slot);
        const float r = 1.0f / sqrtf(s[0] * inv_c + eps);
        if (threadIdx.x == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
        for (int a = threadIdx.x * VEC; a < C; a += 1024 * VEC) {
            const nerf::Place<T, false> at(a, C);
            const Row<T> p = nerf::load_piece<false>(xr, at);
            float w[VEC], b[VEC];
            nerf::load_weights<false, T>(weight, w_f32, at, 1.0f, w);
            nerf::load_weights<false, T>(bias, w_f32, at, 0.0f, b);
            Row<T> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.v[j] = (T)fmaf(((float)p.v[j] - mu) * r, w[j], b[j]);
            nerf::store_piece<false>(y + row * C, at, o);
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward
// Every workgroup walks its rows with the column sums of gw and gb in registers and leaves one partial row
// [2][C] (fp32) of them; layernorm_columns_kernel adds the partials in a fixed order: no atomics, the same bits every run.
// A row stays in registers as it was read; h and q are made from it twice (`forget`: the compiler would keep them), which
// costs less than the registers they fill.  Where a row takes more than a wavefront, the next row is on its way while this
// one waits at its barrier.
template <typename T, int TPR, int NV, int BLOCK, bool TINY>
__global__ __launch_bounds__(BLOCK) void layernorm_bwd_kernel(const T *__restrict__ g_out, int64_t g_stride,
                                                              const T *__restrict__ x, int64_t x_stride, int64_t M, int C,
                                                              const void *__restrict__ weight, int w_f32,
                                                              const float *__restrict__ mean,
                                                              const float *__restrict__ rstd, T *__restrict__ g_x,
                                                              float *__restrict__ partial) {
    constexpr int VEC = Row<T>::VEC, RPB = BLOCK / TPR, LANES = TPR < WAVE ? WAVE : TPR;
    constexpr bool HOIST = NV * VEC <= 8, TOGETHER = TPR > WAVE, AHEAD = TOGETHER && X_AHEAD;
    __shared__ float red[TPR > WAVE ? 2 * 2 * (BLOCK / WAVE) : 1];
    __shared__ float cols[BLOCK > LANES ? 2 * TPR * NV * VEC : 1];
    int slot = 0;
    const int lane = threadIdx.x % TPR;
    const float inv_c = 1.0f / (float)C;
    float w[HOIST ? NV : 1][VEC];
    if constexpr (HOIST) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            nerf::load_weights<TINY, T>(weight, w_f32, nerf::Place<T, TINY>((i * TPR + lane) * VEC, C), 1.0f, w[i]);
    }
    float gw[NV][VEC] = {}, gb[NV][VEC] = {};
    Row<T> px[NV], pg[NV];
    float mu, r;
    auto fetch = [&](int64_t row) {
        mu = mean[row];
        r = rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * TPR + lane) * VEC, C);
            px[i] = nerf::load_piece<TINY>(x + row * x_stride, at);
            pg[i] = nerf::load_piece<TINY>(g_out + row * g_stride, at);
        }
    };
    const int64_t first = (int64_t)blockIdx.x * RPB, step = (int64_t)gridDim.x * RPB;
    const int group = nerf::lane_group<TPR>();
    if (AHEAD) fetch(first + group < M ? first + group : M - 1);
    // (a group beyond the last row goes along to the barriers, with the last row once more and nothing to show for it)
    for (int64_t base = first; base < M; base += step) {
        const bool live = base + group < M;
        const int64_t row = live ? base + group : M - 1;
        if (!TOGETHER && !live) break;
        if (!AHEAD) fetch(row);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * TPR + lane) * VEC, C);
            if constexpr (!HOIST) nerf::load_weights<TINY, T>(weight, w_f32, at, 1.0f, w[0]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float g = (float)pg[i].v[j], h = ((float)px[i].v[j] - mu) * r;
                const float q = at.own(j) ? g * w[HOIST ? i : 0][j] : 0.0f;
                gw[i][j] = !TOGETHER || live ? fmaf(g, h, gw[i][j]) : gw[i][j];
                gb[i][j] += !TOGETHER || live ? g : 0.0f;
                s[0] += q;
                s[1] = at.own(j) ? fmaf(q, h, s[1]) : s[1];
            }
        }
        Row<T> x_now[NV], g_now[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x_now[i] = px[i];
            g_now[i] = pg[i];
            if (!HOIST) { forget(x_now[i]); forget(g_now[i]); }
        }
        const float mu_now = mu, r_now = r;
        if (AHEAD && base + step < M) fetch(base + step + group < M ? base + step + group : M - 1);
        row_sum<TPR, 2, BLOCK>(s, red, slot);
        const float c0 = s[0] * inv_c, c1 = s[1] * inv_c;
        const void *w_again = weight;
        if (!HOIST) asm volatile("" : "+s"(w_again));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * TPR + lane) * VEC, C);
            if constexpr (!HOIST) nerf::load_weights<TINY, T>(w_again, w_f32, at, 1.0f, w[0]);
            Row<T> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float q = (float)g_now[i].v[j] * w[HOIST ? i : 0][j], h = ((float)x_now[i].v[j] - mu_now) * r_now;
                o.v[j] = (T)(r_now * (q - fmaf(h, c1, c0)));
            }
            if (!TOGETHER || live) nerf::store_piece<TINY>(g_x + row * C, at, o);
        }
    }
    if (!partial) return;
    float *dst = partial + (int64_t)blockIdx.x * 2 * C;
    if constexpr (BLOCK == TPR) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * TPR + lane) * VEC, C);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (at.own(j)) { dst[at.at + j] = gw[i][j]; dst[C + at.at + j] = gb[i][j]; }
        }
    } else {
        // lane groups of a wavefront first, then group after group through LDS
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
#pragma unroll
                for (int d = TPR; d < WAVE; d <<= 1) {
                    gw[i][j] += __shfl_xor(gw[i][j], d, WAVE);
                    gb[i][j] += __shfl_xor(gb[i][j], d, WAVE);
                }
        for (int k = 0; k < BLOCK / LANES; ++k) {
            if ((int)threadIdx.x / LANES == k && (int)threadIdx.x % LANES < TPR) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        float *c = cols + (i * VEC + j) * 2 * TPR + lane;
                        c[0] = k ? c[0] + gw[i][j] : gw[i][j];
                        c[TPR] = k ? c[TPR] + gb[i][j] : gb[i][j];
                    }
            }
            __syncthreads();
        }
        for (int k = threadIdx.x; k < TPR * NV * VEC; k += BLOCK) {
            const int l = k % TPR, ij = k / TPR, j = ij % VEC;
            const nerf::Place<T, TINY> at(((ij / VEC) * TPR + l) * VEC, C);
            if (at.own(j)) {
                dst[at.at + j] = cols[ij * 2 * TPR + l];
                dst[C + at.at + j] = cols[ij * 2 * TPR + TPR + l];
            }
        }
    }
}

// out[c] = sum over the G partial rows of column c: 16 columns x 64 slices of the partial rows per workgroup
template <typename W>
__global__ __launch_bounds__(1024) void layernorm_columns_kernel(const float *__restrict__ partial, int G, int64_t C,
                                                                 W *__restrict__ g_weight, W *__restrict__ g_bias) {
    __shared__ float part[64][17];
    const int c = threadIdx.x & 15, s = threadIdx.x >> 4;
    const int64_t at = (int64_t)blockIdx.x * 16 + c;
    float sum = 0.0f;
    if (at < 2 * C) {
#pragma unroll 8
        for (int k = s; k < G; k += 64) sum += partial[(int64_t)k * 2 * C + at];
    }
    part[s][c] = sum;
    __syncthreads();
    if (s < 8) {
        sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += part[s * 8 + k][c];
    }
    __syncthreads();
    if (s < 8) part[s][c] = sum;
    __syncthreads();
    if (s == 0 && at < 2 * C) {
        sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += part[k][c];
        if (at < C ? g_weight != nullptr : g_bias != nullptr) *(at < C ? g_weight + at : g_bias + (at - C)) = (W)sum;
    }
}

// Rows longer than a workgroup's registers: gx in two sweeps, the column sums in a launch of their own.
template <typename T>
__global__ __launch_bounds__(1024) void layernorm_bwd_long_kernel(const T *__restrict__ g_out, int64_t g_stride,
                                                                  const T *__restrict__ x, int64_t x_stride, int64_t M,
                                                                  int C, const void *__restrict__ weight, int w_f32,
                                                                  const float *__restrict__ mean,
                                                                  const float *__restrict__ rstd, T *__restrict__ g_x) {
    constexpr int VEC = Row<T>::VEC;
    __shared__ float red[2 * 2 * 16];
    int slot = 0;
    const float inv_c = (float)(1.0 / (double)C);
    for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
        const T *xr = x + row * x_stride, *gr = g_out + row * g_stride;
        const float mu = mean[row], r = rstd[row];
        float s[2] = {0.0f, 0.0f};
        for (int a = threadIdx.x * VEC; a < C; a += 1024 * VEC) {
            const nerf::Place<T, false> at(a, C);
            const Row<T> px = nerf::load_piece<false>(xr, at), pg = nerf::load_piece<false>(gr, at);
            float w[VEC];
            nerf::load_weights<false, T>(weight, w_f32, at, 1.0f, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float q = (float)pg.v[j] * w[j];
                s[0] += at.own(j) ? q : 0.0f;
                s[1] = at.own(j) ? fmaf(q, ((float)px.v[j] - mu) * r, s[1]) : s[1];
            }
        }
        row_sum<1024, 2, 1024>(s, red, slot);
        const float c0 = s[0] * inv_c, c1 = s[1] * inv_c;
        for (int a = threadIdx.x * VEC; a < C; a += 1024 * VEC) {
            const nerf::Place<T, false> at(a, C);
            const Row<T> px = nerf::load_piece<false>(xr, at), pg = nerf::load_piece<false>(gr, at);
            float w[VEC];
            nerf::load_weights<false, T>(weight, w_f32, at, 1.0f, w);
            Row<T> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                o.v[j] = (T)(r * ((float)pg.v[j] * w[j] - fmaf(((float)px.v[j] - mu) * r, c1, c0)));
            nerf::store_piece<false>(g_x + row * C, at, o);
        }
    }
}

// column sums of `rows` rows per blockIdx.y, one piece of columns per thread
template <typename T>
__global__ __launch_bounds__(256) void layernorm_bwd_long_columns_kernel(const T *__restrict__ g_out, int64_t g_stride,
                                                                         const T *__restrict__ x, int64_t x_stride,
                                                                         int64_t M, int C,
                                                                         const float *__restrict__ mean,
                                                                         const float *__restrict__ rstd,
                                                                         float *__restrict__ partial) {
    constexpr int VEC = Row<T>::VEC;
    const nerf::Place<T, false> at((blockIdx.x * 256 + threadIdx.x) * VEC, C);
    if (!at.live()) return;
    float gw[VEC] = {}, gb[VEC] = {};
    for (int64_t row = blockIdx.y; row < M; row += gridDim.y) {
        const Row<T> px = nerf::load_piece<false>(x + row * x_stride, at);
        const Row<T> pg = nerf::load_piece<false>(g_out + row * g_stride, at);
        const float mu = mean[row], r = rstd[row];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            gw[j] = fmaf((float)pg.v[j], ((float)px.v[j] - mu) * r, gw[j]);
            gb[j] += (float)pg.v[j];
        }
    }
    float *dst = partial + (int64_t)blockIdx.y * 2 * C + at.at;
#pragma unroll
    for (int j = 0; j < VEC; ++j)
        if (at.own(j)) { dst[j] = gw[j]; dst[C + j] = gb[j]; }
}

// ------------------------------------------------------------------------------------------------ launches
constexpr int MAX_REGISTER_ROW = 16384;

// f(TPR, NV, BLOCK, TINY) where TPR lanes of NV pieces hold a row of C values
#define LN_CASE(tpr, values, block, ...)                                                                     \
    if (C <= (int64_t)(tpr) * (values)) {                                                                    \
        constexpr int TPR = (tpr), NV = (values) / Row<T>::VEC, BLOCK = (block);                             \
        constexpr bool TINY = false;                                                                         \
        __VA_ARGS__;                                                                                         \
    }
#define LN_TINY(block, ...)                                                                                  \
    if (C < Row<T>::VEC) {                                                                                   \
        constexpr int TPR = 1, NV = 1, BLOCK = (block);                                                      \
        constexpr bool TINY = true;                                                                          \
        __VA_ARGS__;                                                                                         \
    }
// The smallest lane group that holds a row with one piece a lane; then one wavefront with up to 64 values a lane, which
// needs no barrier; then a workgroup.  Few rows take the workgroup earlier: a row's latency counts, not the barriers.
#define LN_SHORT(block, ...)                                                                                 \
    LN_TINY(block, __VA_ARGS__) else LN_CASE(4, Row<T>::VEC, block, __VA_ARGS__)                             \
    else LN_CASE(8, Row<T>::VEC, block, __VA_ARGS__) else LN_CASE(16, Row<T>::VEC, block, __VA_ARGS__)       \
    else LN_CASE(32, Row<T>::VEC, block, __VA_ARGS__) else LN_CASE(64, Row<T>::VEC, block, __VA_ARGS__)
#define LN_FORWARD(...)                                                                                      \
    LN_SHORT(256, __VA_ARGS__) else LN_CASE(64, 16, 256, __VA_ARGS__)                                        \
    else if (M >= 1024 && C <= 4096) {                                                                       \
        LN_CASE(64, 24, 256, __VA_ARGS__) else LN_CASE(64, 32, 256, __VA_ARGS__)                             \
        else LN_CASE(64, 48, 256, __VA_ARGS__) else LN_CASE(64, 64, 256, __VA_ARGS__)                        \
    }                                                                                                        \
    else LN_CASE(256, 8, 256, __VA_ARGS__) else LN_CASE(256, 16, 256, __VA_ARGS__)                           \
    else LN_CASE(512, 16, 512, __VA_ARGS__) else LN_CASE(1024, 16, 1024, __VA_ARGS__)

// Backward: workgroups as large as the registers of a CU allow, so that few partial rows are left.
#define LN_BACKWARD(...)                                                                                     \
    LN_SHORT(1024, __VA_ARGS__) else LN_CASE(64, 8, 1024, __VA_ARGS__) else LN_CASE(64, 16, 512, __VA_ARGS__) \
    else LN_CASE(256, 8, 1024, __VA_ARGS__) else LN_CASE(256, 16, 1024, __VA_ARGS__)                         \
    else LN_CASE(512, 16, 1024, __VA_ARGS__) else LN_CASE(1024, 16, 1024, __VA_ARGS__)

// partial rows of the weight's gradient: one per workgroup of the backward pass
int backward_groups(int64_t M, int64_t C) {
    const int64_t per = C <= 512 ? 16 : C <= 1024 ? 8 : C <= 4096 ? 4 : C <= 8192 ? 2 : 1;      // rows a workgroup takes at once, at least
    const int64_t g = (M + per - 1) / per, most = C > MAX_REGISTER_ROW ? 32 : C <= 1024 ? 512 : 256;
    return (int)(g < 1 ? 1 : g > most ? most : g);
}

template <typename T>
void launch_forward(const void *x, int64_t x_stride, int64_t M, int64_t C, const void *weight, const void *bias, int w_f32,
                    float eps, void *y, float *mean, float *rstd, hipStream_t stream) {
    const T *xt = static_cast<const T *>(x);
    T *yt = static_cast<T *>(y);
    if (C > MAX_REGISTER_ROW) {
        hipLaunchKernelGGL(layernorm_long_kernel<T>, dim3((unsigned)(M < 4096 ? M : 4096)), dim3(1024), 0, stream, xt,
                           x_stride, M, (int)C, weight, bias, w_f32, eps, yt, mean, rstd);
        return;
    }
    LN_FORWARD({
        int64_t grid = (M + BLOCK / TPR - 1) / (BLOCK / TPR);
        if (grid > 256 * 8) grid = 256 * 8;
        hipLaunchKernelGGL((layernorm_kernel<T, TPR, NV, BLOCK, TINY>), dim3((unsigned)grid), dim3(BLOCK), 0, stream, xt, x_stride,
                           M, (int)C, weight, bias, w_f32, eps, yt, mean, rstd);
    })
}

template <typename T>
void launch_backward(const void *g_out, int64_t g_stride, const void *x, int64_t x_stride, int64_t M, int64_t C,
                     const void *weight, int w_f32, const float *mean, const float *rstd, void *g_x, void *g_weight,
                     void *g_bias, float *partial, hipStream_t stream) {
    const T *xt = static_cast<const T *>(x), *gt = static_cast<const T *>(g_out);
    T *gx = static_cast<T *>(g_x);
    const int G = backward_groups(M, C);
    const bool columns = g_weight || g_bias;
    if (M > 0 && C > MAX_REGISTER_ROW) {
        hipLaunchKernelGGL(layernorm_bwd_long_kernel<T>, dim3((unsigned)(M < 4096 ? M : 4096)), dim3(1024), 0, stream, gt,
                           g_stride, xt, x_stride, M, (int)C, weight, w_f32, mean, rstd, gx);
        if (columns)
            hipLaunchKernelGGL(layernorm_bwd_long_columns_kernel<T>,
                               dim3((unsigned)((C + 256 * Row<T>::VEC - 1) / (256 * Row<T>::VEC)), G), dim3(256), 0, stream,
                               gt, g_stride, xt, x_stride, M, (int)C, mean, rstd, partial);
    } else if (M > 0) {
        LN_BACKWARD({
            hipLaunchKernelGGL((layernorm_bwd_kernel<T, TPR, NV, BLOCK, TINY>), dim3(G), dim3(BLOCK), 0, stream, gt, g_stride, xt,
                               x_stride, M, (int)C, weight, w_f32, mean, rstd, gx, columns ? partial : nullptr);
        })
    }
    if (columns) {
        const unsigned grid = (unsigned)((2 * C + 15) / 16);
        const int rows = M > 0 ? G : 0;
        if (w_f32)
            hipLaunchKernelGGL(layernorm_columns_kernel<float>, dim3(grid), dim3(1024), 0, stream, partial, rows, C,
                               static_cast<float *>(g_weight), static_cast<float *>(g_bias));
        else
            hipLaunchKernelGGL(layernorm_columns_kernel<T>, dim3(grid), dim3(1024), 0, stream, partial, rows, C,
                               static_cast<T *>(g_weight), static_cast<T *>(g_bias));
    }
}

bool sizes_ok(int64_t M, int64_t C) { return M >= 0 && C >= 1 && C <= (int64_t)1 << 30 && M <= INT64_MAX / 8 / C; }

}  // namespace

NERF_API int nerf_layernorm(const void *x, int64_t x_stride, int dtype, int64_t M, int64_t C, const void *weight,
                            const void *bias, int w_dtype, double eps, void *y, float *mean, float *rstd,
                            nerf_stream_t stream) {
    NERF_REQUIRE(nerf::known_dtype(dtype), "nerf_layernorm: unknown dtype");
    NERF_REQUIRE(w_dtype == dtype || w_dtype == NERF_F32, "nerf_layernorm: weights are of x's dtype or fp32");
    NERF_REQUIRE(sizes_ok(M, C), "nerf_layernorm: size out of range");
    NERF_REQUIRE(eps >= 0.0 && eps < 1e30, "nerf_layernorm: eps must be finite and >= 0");
    if (M == 0) return NERF_OK;
    NERF_REQUIRE(x && y, "nerf_layernorm: null pointer");
    NERF_REQUIRE(x_stride >= (M > 1 ? C : 0), "nerf_layernorm: rows overlap (x_stride < C)");
    NERF_FOR_DTYPE(dtype, T, launch_forward<T>(x, x_stride, M, C, weight, bias, w_dtype == NERF_F32, (float)eps, y, mean,
                                               rstd, nerf::as_stream(stream)));
    return nerf::check_launch("nerf_layernorm");
}

NERF_API int64_t nerf_layernorm_backward_workspace_bytes(int64_t M, int64_t C) {
    if (!sizes_ok(M, C)) return nerf::fail(NERF_ERR_ARG, "nerf_layernorm_backward_workspace_bytes: size out of range"), -1;
    return (int64_t)backward_groups(M, C) * 2 * C * 4;
}

NERF_API int nerf_layernorm_backward(const void *g_out, int64_t g_stride, const void *x, int64_t x_stride, int dtype, int64_t M,
                                     int64_t C, const void *weight, int w_dtype, const float *mean, const float *rstd,
                                     void *g_x, void *g_weight, void *g_bias, void *workspace, nerf_stream_t stream) {
    NERF_REQUIRE(nerf::known_dtype(dtype), "nerf_layernorm_backward: unknown dtype");
    NERF_REQUIRE(w_dtype == dtype || w_dtype == NERF_F32, "nerf_layernorm_backward: weights are of x's dtype or fp32");
    NERF_REQUIRE(sizes_ok(M, C), "nerf_layernorm_backward: size out of range");
    NERF_REQUIRE(M == 0 || (g_out && x && mean && rstd && g_x), "nerf_layernorm_backward: null pointer");
    NERF_REQUIRE(!(g_weight || g_bias) || M == 0 || workspace, "nerf_layernorm_backward: workspace missing");
    NERF_REQUIRE(M <= 1 || (x_stride >= C && g_stride >= C), "nerf_layernorm_backward: rows overlap (stride < C)");
    NERF_FOR_DTYPE(dtype, T, launch_backward<T>(g_out, g_stride, x, x_stride, M, C, weight, w_dtype == NERF_F32, mean, rstd,
                                                g_x, g_weight, g_bias, static_cast<float *>(workspace),
                                                nerf::as_stream(stream)));
    return nerf::check_launch("nerf_layernorm_backward");
}
