// Layer norm over the last axis, forward and backward, with the reduction of the weight's and the bias's gradient.
//
//   y = (x - mu) r w + b,   mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps)
//   gx = r (q - mean(q) - h mean(q h)),  q = g w, h = (x - mu) r;   gw = sum_rows g h,   gb = sum_rows g
//
// A row stays in registers between its one read and its one write: TPR lanes hold it as NV 16-byte pieces each.  Statistics
// and sums are fp32, and an offset of the row costs no digits.  The first mean m, from the sum of x, is off by some roundings
// of the offset's size, which may be larger than the deviations; the second sums are of d = x - m and of d^2, and with e = mean(d)
//   mu = m + e,   var = mean(d^2) - e^2,   (x - mu) r = d r - e r
// are off by roundings of the deviations' size.  Where m is smaller than the deviations it is no worse than m + e, and e is
// taken as 0.  Where it is so much larger that e^2 is not small beside var (constant rows), d - e is summed once more in
// place of d.  (mu itself is stored as fp32, and that is what the backward pass takes.)
// Rows of up to 64 lanes need no barrier; a longer row takes several wavefronts.
//
// Bound by HBM.  Forward 262144 x 256 fp32: 90 us, 6.0 TB/s read + written (a copy of that size: 5.4); 16384 x 2048 bf16
// 28 us (4.8); 8192 x 4096 fp32 46 us (5.8); 1 row of 4096: 2.8 us.  Backward 786432 x 256 fp32: 455 + 12 us for the columns,
// 5.2 TB/s; 8192 x 4096 bf16: 40 + 5 us, 4.5 TB/s.  Where it is not:
// - rows of 8193..16384 values: a workgroup holds one row, in lockstep.  As 2048 x 16384 bf16 the values of 8192 x 4096 take 35 us
//   forward instead of 26 and 66 + 13 backward instead of 40 + 5 (fp32: 62 instead of 46, 105 + 13 instead of 76 + 5, with 9
//   registers spilled);
// - longer rows, which are read three times by one workgroup each: 1024 x 32768 36 us forward and 54 + 25 + 10 backward in bf16,
//   83 and 100 + 48 + 10 in fp32; few and very long ones do not fill the chip (256 x 131072 fp32: 99 and 110 + 54 + 38 us);
// - rows of fewer than 8 16-bit or 4 fp32 values, which go value by value: 11000000 x 3 fp32 76 us forward (3.5 TB/s) and 103 + 5
//   backward (3.7), 4800000 x 7 bf16 76 (1.8) and 101 + 5 (1.9).
#include "rows.h"

namespace {

using nerf::Row;

// Rows of at most one wavefront's registers: TPR <= 64 lanes share one.  Wider rows take `waves` wavefronts each (WIDE), as
// many as the row needs, and a workgroup a whole number of such groups.
//
// Sum of K values over the lanes that share a row.  WIDE: through LDS, all groups of the workgroup at once; `slot`
// alternates so that one barrier per sum is enough (a wave that runs ahead writes the other half of `red`).
constexpr int MAX_WAVES = 16;

template <int TPR, bool WIDE, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float *red, int &slot, int waves) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = nerf::lane_sum<TPR>(v[k]);
    if constexpr (WIDE) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
        float *r = red + slot * 2 * MAX_WAVES;                // (the same halves for one value and for two)
        static_assert(K <= 2, "red");
        slot ^= 1;
        if ((threadIdx.x & (WAVE - 1)) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) r[wave * K + k] = v[k];
        }
        __syncthreads();
        const int w = threadIdx.x & (MAX_WAVES - 1);
        r += (wave / waves * waves + (w < waves ? w : 0)) * K;
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = nerf::lane_sum<MAX_WAVES>(w < waves ? r[k] : 0.0f);
    }
}

// Which of its row's lanes a thread is, and which row of its workgroup's (a scalar where a wavefront has one row).
template <int TPR, bool WIDE>
struct Lanes {
    int lane, group, width;
    __device__ __forceinline__ explicit Lanes(int waves) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
        if (WIDE) {
            group = wave / waves;
            lane = (int)threadIdx.x - group * waves * WAVE;
            width = waves * WAVE;
        } else {
            group = TPR == WAVE ? wave : (int)threadIdx.x / TPR;
            lane = threadIdx.x % TPR;
            width = TPR;
        }
    }
};

// The compiler may not keep what it made of p (or loaded through p) before this point.
template <typename T>
__device__ __forceinline__ void forget(Row<T> &p) {
    uint32_t u[4];
    __builtin_memcpy(u, &p, 16);
    asm volatile("" : "+v"(u[0]), "+v"(u[1]), "+v"(u[2]), "+v"(u[3]));
    __builtin_memcpy(&p, u, 16);
}

// From the sums of d and of d^2, d = x - m: e = mean(d) where that improves m, and r.  (A NaN stays one, an infinity too.)
struct Moments {
    float e, r;
    __device__ __forceinline__ Moments(const float (&sums)[2], float m, float inv_c, float eps) {
        const float square = sums[1] * inv_c;
        e = m * m > square ? sums[0] * inv_c : 0.0f;
        const float var = fmaf(-e, e, square);
        r = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps);
    }
};

// The sums are to be taken again, about m + e: m is 2^10 deviations or more.  (28 roundings take m off by 2^-19 of itself, by 2^-9
// of a deviation where this says no: e^2 is 2^-18 of the variance.  A row of C > 16384 values takes C / 1024 of them more, one
// of 2^24 up to 2^-10: e^2 is then the variance's size at the worst.)  The same for all lanes that share a row.
__device__ __forceinline__ bool far_off(const float (&sums)[2], float m, float inv_c) { return m * m > 0x1p20f * (sums[1] * inv_c); }

template <typename T, int TPR, int NV, bool WIDE, bool TINY>
__global__ __launch_bounds__(WIDE ? 1024 : 256) void layernorm_kernel(const T *__restrict__ x, int64_t x_stride, int64_t M, int C,
                                                          const void *__restrict__ weight, const void *__restrict__ bias,
                                                          int w_f32, float eps, T *__restrict__ y,
                                                          float *__restrict__ mean, float *__restrict__ rstd, int waves, int64_t per) {
    constexpr int VEC = Row<T>::VEC;
    constexpr bool HOIST = NV * VEC <= 8;                     // the weights stay in registers from row to row
    __shared__ float red[WIDE ? 2 * 2 * MAX_WAVES : 1];
    int slot = 0;
    const Lanes<TPR, WIDE> at_row(waves);                     // (WIDE: one row a workgroup)
    const int lane = at_row.lane, width = at_row.width;
    const int64_t rows = WIDE ? 1 : 256 / TPR;
    const float inv_c = 1.0f / (float)C;
    float w[HOIST ? NV : 1][VEC], b[HOIST ? NV : 1][VEC];
    if constexpr (HOIST) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * width + lane) * VEC, C);
            nerf::load_weights<TINY, T>(weight, w_f32, at, 1.0f, w[i]);
            nerf::load_weights<TINY, T>(bias, w_f32, at, 0.0f, b[i]);
        }
    }
    const int64_t begin = (int64_t)blockIdx.x * per * rows, end = begin + per * rows < M ? begin + per * rows : M;
    for (int64_t row = begin + at_row.group; row < end; row += rows) {
        float v[NV][VEC], s[1] = {0.0f}, t[2];
        Row<T> p[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            p[i] = nerf::load_piece<TINY>(x + row * x_stride, nerf::Place<T, TINY>((i * width + lane) * VEC, C));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * width + lane) * VEC, C);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                v[i][j] = (float)p[i].v[j];
                s[0] += at.own(j) ? v[i][j] : 0.0f;
            }
        }
        row_sum<TPR, WIDE, 1>(s, red, slot, waves);
        float m = s[0] * inv_c;
        auto about = [&](float shift) {                       // v -= shift; t <- the sums of v and v^2
            t[0] = t[1] = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const nerf::Place<T, TINY> at((i * width + lane) * VEC, C);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    v[i][j] -= shift;
                    const float d = at.own(j) ? v[i][j] : 0.0f;
                    t[0] += d;
                    t[1] = fmaf(d, d, t[1]);
                }
            }
            row_sum<TPR, WIDE, 2>(t, red, slot, waves);
        };
        about(m);
        if (far_off(t, m, inv_c)) {
            const float e = t[0] * inv_c;
            m += e;
            about(e);
        }
        const Moments stat(t, m, inv_c, eps);
        const float r = stat.r, shift = -stat.e * r;
        if (lane == 0) {
            if (mean) mean[row] = m + stat.e;
            if (rstd) rstd[row] = r;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * width + lane) * VEC, C);
            if constexpr (!HOIST) {
                nerf::load_weights<TINY, T>(weight, w_f32, at, 1.0f, w[0]);
                nerf::load_weights<TINY, T>(bias, w_f32, at, 0.0f, b[0]);
            }
            Row<T> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) o.v[j] = (T)fmaf(fmaf(v[i][j], r, shift), w[HOIST ? i : 0][j], b[HOIST ? i : 0][j]);
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
    __shared__ float red[2 * 2 * MAX_WAVES];
    int slot = 0;
    const float inv_c = (float)(1.0 / (double)C);
    for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
        const T *xr = x + row * x_stride;
        float s[1] = {0.0f}, t[2];
        for (int a = threadIdx.x * VEC; a < C; a += 1024 * VEC) {
            const nerf::Place<T, false> at(a, C);
            const Row<T> p = nerf::load_piece<false>(xr, at);
#pragma unroll
            for (int j = 0; j < VEC; ++j) s[0] += at.own(j) ? (float)p.v[j] : 0.0f;
        }
        row_sum<WAVE, true, 1>(s, red, slot, MAX_WAVES);
        const float m = s[0] * inv_c;
        float e = 0.0f;
        auto about = [&] {                                    // t <- the sums of d = x - m - e and of d^2
            t[0] = t[1] = 0.0f;
            for (int a = threadIdx.x * VEC; a < C; a += 1024 * VEC) {
                const nerf::Place<T, false> at(a, C);
                const Row<T> p = nerf::load_piece<false>(xr, at);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float d = at.own(j) ? ((float)p.v[j] - m) - e : 0.0f;
                    t[0] += d;
                    t[1] = fmaf(d, d, t[1]);
                }
            }
            row_sum<WAVE, true, 2>(t, red, slot, MAX_WAVES);
        };
        about();
        if (far_off(t, m, inv_c)) {
            e = t[0] * inv_c;
            about();
        }
        const Moments stat(t, m, inv_c, eps);
        const float r = stat.r, shift = -stat.e * r;
        if (threadIdx.x == 0) {
            if (mean) mean[row] = m + (e + stat.e);
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
            for (int j = 0; j < VEC; ++j) o.v[j] = (T)fmaf(fmaf(((float)p.v[j] - m) - e, r, shift), w[j], b[j]);
            nerf::store_piece<false>(y + row * C, at, o);
        }
    }
}

// ------------------------------------------------------------------------------------------------ backward
template <typename T>
__device__ __forceinline__ void store_column(void *out, int f32, int c, float v) {
    if (f32)
        static_cast<float *>(out)[c] = v;
    else
        static_cast<T *>(out)[c] = (T)v;
}

// Every workgroup walks its rows with the column sums of gw and gb in registers and leaves one partial row
// [2][C] (fp32) of them; layernorm_columns_kernel adds the partials in a fixed order: no atomics, the same bits every run.
// A row stays in registers as it was read; h and q are made from it twice (`forget`: the compiler would keep them), which
// costs less than the registers they fill.  Where a row takes more than a wavefront, the next row is on its way while this
// one waits at its barrier.
template <typename T, int TPR, int NV, bool WIDE, bool TINY>
__global__ __launch_bounds__(1024) void layernorm_bwd_kernel(const T *__restrict__ g_out, int64_t g_stride,
                                                              const T *__restrict__ x, int64_t x_stride, int64_t M, int C,
                                                              const void *__restrict__ weight, int w_f32,
                                                              const float *__restrict__ mean,
                                                              const float *__restrict__ rstd, T *__restrict__ g_x,
                                                              float *__restrict__ partial, void *__restrict__ g_weight,
                                                              void *__restrict__ g_bias, int waves, int64_t per) {
    constexpr int VEC = Row<T>::VEC;
    constexpr bool HOIST = NV * VEC <= 8, AHEAD = WIDE && NV * VEC <= 8;
    __shared__ float red[WIDE ? 2 * 2 * MAX_WAVES : 1];
    extern __shared__ float cols[];                           // the groups' column sums
    int slot = 0;
    const Lanes<TPR, WIDE> at_row(waves);
    const int lane = at_row.lane, width = at_row.width, group = at_row.group;
    const int lanes = WIDE ? width : WAVE, groups = blockDim.x / lanes, rows = blockDim.x / width;
    const float inv_c = 1.0f / (float)C;
    float w[HOIST ? NV : 1][VEC];
    if constexpr (HOIST) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            nerf::load_weights<TINY, T>(weight, w_f32, nerf::Place<T, TINY>((i * width + lane) * VEC, C), 1.0f, w[i]);
    }
    float gw[NV][VEC] = {}, gb[NV][VEC] = {};
    Row<T> px[NV], pg[NV];
    float mu, r;
    auto fetch = [&](int64_t row) {
        mu = mean[row];
        r = rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * width + lane) * VEC, C);
            px[i] = nerf::load_piece<TINY>(x + row * x_stride, at);
            pg[i] = nerf::load_piece<TINY>(g_out + row * g_stride, at);
        }
    };
    // per > 0: so many steps of rows next to each other; 0: every gridDim.x-th step
    const int64_t first = (int64_t)blockIdx.x * (per ? per : 1) * rows, step = per ? rows : (int64_t)gridDim.x * rows;
    const int64_t end = per && first + per * rows < M ? first + per * rows : M;
    if (AHEAD) fetch(first + group < end ? first + group : end - 1);
    // (a group beyond the last row goes along to the barriers, with the last row once more and nothing to show for it)
    for (int64_t base = first; base < end; base += step) {
        const bool live = base + group < end;
        const int64_t row = live ? base + group : end - 1;
        if (!WIDE && !live) break;
        if (!AHEAD) fetch(row);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * width + lane) * VEC, C);
            if constexpr (!HOIST) nerf::load_weights<TINY, T>(weight, w_f32, at, 1.0f, w[0]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float g = (float)pg[i].v[j], h = ((float)px[i].v[j] - mu) * r;
                const float q = at.own(j) ? g * w[HOIST ? i : 0][j] : 0.0f;
                gw[i][j] = !WIDE || live ? fmaf(g, h, gw[i][j]) : gw[i][j];
                gb[i][j] += !WIDE || live ? g : 0.0f;
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
        if (AHEAD && base + step < end) fetch(base + step + group < end ? base + step + group : end - 1);
        row_sum<TPR, WIDE, 2>(s, red, slot, waves);
        const float c0 = s[0] * inv_c, c1 = s[1] * inv_c;
        const void *w_again = weight;
        if (!HOIST) asm volatile("" : "+s"(w_again));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * width + lane) * VEC, C);
            if constexpr (!HOIST) nerf::load_weights<TINY, T>(w_again, w_f32, at, 1.0f, w[0]);
            Row<T> o;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float q = (float)g_now[i].v[j] * w[HOIST ? i : 0][j], h = ((float)x_now[i].v[j] - mu_now) * r_now;
                o.v[j] = (T)(r_now * (q - fmaf(h, c1, c0)));
            }
            if (!WIDE || live) nerf::store_piece<TINY>(g_x + row * C, at, o);
        }
    }
    if (!g_weight && !g_bias) return;
    // one workgroup alone has the gradients themselves
    auto put = [&](int c, float sum, bool bias) {
        void *out = bias ? g_bias : g_weight;
        if (gridDim.x > 1)
            partial[((int64_t)blockIdx.x * 2 + (bias ? 1 : 0)) * C + c] = sum;
        else if (out)
            store_column<T>(out, w_f32, c, sum);
    };
    // lane groups of a wavefront first, then the groups of the workgroup through LDS, in order
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j)
#pragma unroll
            for (int d = TPR; d < WAVE; d <<= 1) {
                gw[i][j] += __shfl_xor(gw[i][j], d, WAVE);
                gb[i][j] += __shfl_xor(gb[i][j], d, WAVE);
            }
    if (groups == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const nerf::Place<T, TINY> at((i * width + lane) * VEC, C);
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (at.own(j)) { put(at.at + j, gw[i][j], false); put(at.at + j, gb[i][j], true); }
        }
        return;
    }
    // gw, then gb: [group][NV * VEC][width]
    const int mine = threadIdx.x / lanes, size = NV * VEC * width;
    const bool has = (int)threadIdx.x - mine * lanes < width;
    auto join = [&](const float (&v)[NV][VEC], bool bias) {
        __syncthreads();
        if (has) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) cols[mine * size + (i * VEC + j) * width + lane] = v[i][j];
        }
        __syncthreads();
        for (int k = threadIdx.x; k < size; k += blockDim.x) {
            const int l = k % width, ij = k / width, j = ij % VEC;
            const nerf::Place<T, TINY> at(((ij / VEC) * width + l) * VEC, C);
            float sum = 0.0f;
            for (int g = 0; g < groups; ++g) sum += cols[g * size + k];
            if (at.own(j)) put(at.at + j, sum, bias);
        }
    };
    join(gw, false);
    join(gb, true);
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
        row_sum<WAVE, true, 2>(s, red, slot, MAX_WAVES);
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
constexpr int MAX_REGISTER_ROW = 16384;      // 1024 threads x 16 values

// f(TPR, NV, WIDE, TINY) where TPR lanes of NV pieces hold a row of C values
#define LN_USE(tpr, nv, wide, tiny, ...)                                                                     \
    {                                                                                                        \
        constexpr int TPR = (tpr), NV = (nv);                                                                \
        constexpr bool WIDE = (wide), TINY = (tiny);                                                         \
        __VA_ARGS__;                                                                                         \
    }
// (fp32 alone: for 16-bit rows the condition in front never holds, and the kernel is not made)
#define LN_USE_F32(tpr, nv, ...)                                                                             \
    {                                                                                                        \
        if constexpr (sizeof(T) == 4) LN_USE(tpr, nv, false, false, __VA_ARGS__)                             \
    }
#define LN_CASE(tpr, nv, ...) if (C <= (int64_t)(tpr) * (nv) * Row<T>::VEC) LN_USE(tpr, nv, false, false, __VA_ARGS__)
// The smallest lane group that holds a row with one piece a lane, then one wavefront with more: no barrier.
#define LN_SHORT(...)                                                                                        \
    if (C < Row<T>::VEC) LN_USE(1, 1, false, true, __VA_ARGS__)                                              \
    else LN_CASE(1, 1, __VA_ARGS__) else LN_CASE(2, 1, __VA_ARGS__) else LN_CASE(4, 1, __VA_ARGS__)          \
    else LN_CASE(8, 1, __VA_ARGS__) else LN_CASE(16, 1, __VA_ARGS__)                                         \
    else LN_CASE(32, 1, __VA_ARGS__) else LN_CASE(64, 1, __VA_ARGS__)

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
    // up to 32 values a lane a wavefront keeps a row to itself; few rows are spread wider, a row's latency counts there
    constexpr int VEC = Row<T>::VEC;
    const bool few = M < 1024;
    // Every workgroup takes its rows once, in the order of the addresses: 1 GB of fp32 rows of 256 at 6.2 TB/s, where 2048
    // workgroups that stride over the rows reach 5.2.  Short 16-bit rows are too little work for that (4.8 TB/s: the
    // weights come first): 4 of them one after another, 5.8 TB/s.
    auto run = [&](auto kernel, int64_t rows, int waves, int64_t in_turn) {
        const int64_t steps = (M + rows - 1) / rows;
        const int threads = waves ? waves * WAVE : 256;
        int64_t per = steps < 4 * 2048 ? 1 : in_turn;
        while ((steps + per - 1) / per * threads > (int64_t)1 << 31) per *= 2;       // a launch's threads are counted in 32 bits
        const int64_t grid = (steps + per - 1) / per;
        hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), 0, stream, xt, x_stride, M, (int)C,
                           weight, bias, w_f32, eps, yt, mean, rstd, waves, per);
    };
#define LN_RUN run(layernorm_kernel<T, TPR, NV, WIDE, TINY>, WIDE ? 1 : 256 / TPR, WIDE ? (int)((C + NV * VEC * WAVE - 1) / (NV * VEC * WAVE)) : 0, NV == 1 && VEC == 8 && !WIDE ? 4 : 1)
    LN_SHORT(LN_RUN) else LN_CASE(64, 2, LN_RUN)
    else if (few && C <= 8 * 1024) LN_USE(64, 8 / VEC, true, false, LN_RUN)
    else LN_CASE(64, 3, LN_RUN) else LN_CASE(64, 4, LN_RUN)
    else if (VEC == 4 && C <= 64 * 24) LN_USE_F32(64, 6, LN_RUN)
    else if (VEC == 4 && C <= 64 * 32) LN_USE_F32(64, 8, LN_RUN)
    else LN_USE(64, 16 / VEC, true, false, LN_RUN)
#undef LN_RUN
}

// How the backward pass walks the rows.
struct Walk {
    int rows, waves, threads;          // of a workgroup: rows at once, wavefronts per row (0: lanes of one), threads
    int64_t groups, per;               // workgroups = partial rows of the weight's gradient; see the kernel
    bool alone;                        // one workgroup, which stores the gradients itself
};

// Workgroups as large as the registers of a CU allow, so that few partial rows are left: as many as the chip holds at once,
// striding over the rows.  Short fp32 rows in large numbers are quicker in the order of the addresses, 16 steps a workgroup
// (786432 x 256: 470 us instead of 500); 16-bit rows are not (239 us instead of 234 at the same bytes).
Walk plan_walk(int64_t M, int64_t C, int dtype) {
    // up to so many steps of one workgroup, a few us each, are quicker than a second launch for the columns
    constexpr int64_t ONE_WORKGROUP = 4, STRIDING = 256, IN_ORDER = 16, IN_ORDER_FROM = 1024, IN_ORDER_MOST = 4096;
    const int vec = 16 / nerf::dtype_bytes(dtype);
    Walk w = {};
    if (C > MAX_REGISTER_ROW) {
        w.groups = M < 1 ? 1 : M > 32 ? 32 : M;              // of layernorm_bwd_long_columns_kernel
        return w;
    }
    if (C <= (dtype == NERF_F32 ? 512 : WAVE * vec)) {
        int lanes = 1;
        while (lanes < WAVE && lanes * vec < C) lanes <<= 1;
        w.rows = 1024 / lanes;
        w.threads = 1024;
    } else {
        const int values = C <= 8 * 1024 ? 8 : 16;
        w.waves = (int)((C + values * WAVE - 1) / (values * WAVE));
        w.rows = MAX_WAVES / w.waves;
        w.threads = w.rows * w.waves * WAVE;
    }
    const int64_t steps = (M + w.rows - 1) / w.rows;
    w.alone = steps <= ONE_WORKGROUP;
    if (w.alone) {
        w.groups = 1;
    } else if (dtype == NERF_F32 && w.waves == 0 && steps >= IN_ORDER * IN_ORDER_FROM) {
        w.per = (steps + IN_ORDER_MOST - 1) / IN_ORDER_MOST;
        if (w.per < IN_ORDER) w.per = IN_ORDER;
        w.groups = (steps + w.per - 1) / w.per;
    } else {
        w.groups = steps < STRIDING ? steps : STRIDING;
    }
    return w;
}

template <typename T>
void launch_backward(const void *g_out, int64_t g_stride, const void *x, int64_t x_stride, int64_t M, int64_t C,
                     const void *weight, int w_f32, const float *mean, const float *rstd, void *g_x, void *g_weight,
                     void *g_bias, float *partial, hipStream_t stream) {
    const T *xt = static_cast<const T *>(x), *gt = static_cast<const T *>(g_out);
    T *gx = static_cast<T *>(g_x);
    const bool columns = g_weight || g_bias;
    constexpr int VEC = Row<T>::VEC;
    const Walk walk = plan_walk(M, C, VEC == 4 ? NERF_F32 : NERF_BF16);
    if (M > 0 && C > MAX_REGISTER_ROW) {
        hipLaunchKernelGGL(layernorm_bwd_long_kernel<T>, dim3((unsigned)(M < 4096 ? M : 4096)), dim3(1024), 0, stream, gt,
                           g_stride, xt, x_stride, M, (int)C, weight, w_f32, mean, rstd, gx);
        if (columns)
            hipLaunchKernelGGL(layernorm_bwd_long_columns_kernel<T>,
                               dim3((unsigned)((C + 256 * VEC - 1) / (256 * VEC)), (unsigned)walk.groups), dim3(256), 0, stream, gt,
                               g_stride, xt, x_stride, M, (int)C, mean, rstd, partial);
    } else if (M > 0) {
        // LDS: the column sums of every group of lanes that has one, where there is more than one group
        auto run = [&](auto kernel, int lanes, int values) {
            const int lds = lanes < walk.threads ? (lanes < WAVE ? walk.threads / WAVE : walk.threads / lanes) * lanes * values * 4 : 0;
            hipLaunchKernelGGL(kernel, dim3((unsigned)walk.groups), dim3(walk.threads), lds, stream, gt, g_stride, xt, x_stride, M,
                               (int)C, weight, w_f32, mean, rstd, gx, partial, g_weight, g_bias, walk.waves,
                               walk.per);
        };
#define LN_RUN run(layernorm_bwd_kernel<T, TPR, NV, WIDE, TINY>, WIDE ? walk.waves * WAVE : TPR, NV * VEC)
        LN_SHORT(LN_RUN)
        else if (VEC == 4 && C <= 64 * 8) LN_USE_F32(64, 2, LN_RUN)
        else if (C <= 8 * 1024) LN_USE(64, 8 / VEC, true, false, LN_RUN)
        else LN_USE(64, 16 / VEC, true, false, LN_RUN)
#undef LN_RUN
    }
    if (columns && !(walk.alone && M > 0)) {
        const unsigned grid = (unsigned)((2 * C + 15) / 16);
        if (w_f32)
            hipLaunchKernelGGL(layernorm_columns_kernel<float>, dim3(grid), dim3(1024), 0, stream, partial, M > 0 ? (int)walk.groups : 0, C,
                               static_cast<float *>(g_weight), static_cast<float *>(g_bias));
        else
            hipLaunchKernelGGL(layernorm_columns_kernel<T>, dim3(grid), dim3(1024), 0, stream, partial, M > 0 ? (int)walk.groups : 0, C,
                               static_cast<T *>(g_weight), static_cast<T *>(g_bias));
    }
}

bool sizes_ok(int64_t M, int64_t C) { return M >= 0 && C >= 1 && C <= (int64_t)1 << 24 && M <= INT64_MAX / 8 / C; }

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

NERF_API int64_t nerf_layernorm_backward_workspace_bytes(int64_t M, int64_t C, int dtype) {
    if (!nerf::known_dtype(dtype) || !sizes_ok(M, C)) return nerf::fail(NERF_ERR_ARG, "nerf_layernorm_backward_workspace_bytes: size out of range"), -1;
    const Walk w = plan_walk(M, C, dtype);
    return w.alone || M == 0 ? 0 : w.groups * 2 * C * 4;
}

NERF_API int nerf_layernorm_backward(const void *g_out, int64_t g_stride, const void *x, int64_t x_stride, int dtype, int64_t M,
                                     int64_t C, const void *weight, int w_dtype, const float *mean, const float *rstd,
                                     void *g_x, void *g_weight, void *g_bias, void *workspace, nerf_stream_t stream) {
    NERF_REQUIRE(nerf::known_dtype(dtype), "nerf_layernorm_backward: unknown dtype");
    NERF_REQUIRE(w_dtype == dtype || w_dtype == NERF_F32, "nerf_layernorm_backward: weights are of x's dtype or fp32");
    NERF_REQUIRE(sizes_ok(M, C), "nerf_layernorm_backward: size out of range");
    NERF_REQUIRE(M == 0 || (g_out && x && mean && rstd && g_x), "nerf_layernorm_backward: null pointer");
    NERF_REQUIRE(!(g_weight || g_bias) || workspace || nerf_layernorm_backward_workspace_bytes(M, C, dtype) == 0,
                 "nerf_layernorm_backward: workspace missing");
    NERF_REQUIRE(M <= 1 || (x_stride >= C && g_stride >= C), "nerf_layernorm_backward: rows overlap (stride < C)");
    NERF_FOR_DTYPE(dtype, T, launch_backward<T>(g_out, g_stride, x, x_stride, M, C, weight, w_dtype == NERF_F32, mean, rstd,
                                                g_x, g_weight, g_bias, static_cast<float *>(workspace),
                                                nerf::as_stream(stream)));
    return nerf::check_launch("nerf_layernorm_backward");
}
