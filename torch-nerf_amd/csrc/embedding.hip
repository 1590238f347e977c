// Embedding lookup with scaling, and its gradient by sorted ids.
//
//   out[i] = scale * table[ids[i]]
//   g_table[v] = scale * sum over { i : ids[i] = v, v != padding_idx } of g_out[i]
//
// An id outside [0, rows) is never used as an address: its output row is NaN, its gradient is dropped.
//
// Gradient: the pairs (id, position) are sorted by id with a stable radix sort, so that the rows of one id stand together
// in the order they came in.  The sorted list is cut into chunks; a lane group walks one chunk with the running sum in
// registers and stores a row of the table when its id ends.  An id that crosses chunks leaves fp32 partial rows, which
// embedding_join_kernel adds in the order of the chunks.  No atomics on values: the same bits every run.
#include "rows.h"

namespace {

using nerf::Row;

__device__ __forceinline__ int64_t load_id(const void *ids, int wide, int64_t i) {
    return wide ? static_cast<const int64_t *>(ids)[i] : (int64_t) static_cast<const int32_t *>(ids)[i];
}

// 2^shift lanes share a row and step through its pieces
template <typename T>
__global__ __launch_bounds__(256) void embedding_kernel(const T *__restrict__ table, int64_t rows, int64_t row_stride,
                                                        int64_t dim, const void *__restrict__ ids, int wide, int64_t n,
                                                        float scale, int shift, T *__restrict__ out) {
    constexpr int VEC = Row<T>::VEC;
    const int per = 256 >> shift, lane = threadIdx.x & ((1 << shift) - 1);
    for (int64_t i = (int64_t)blockIdx.x * per + (threadIdx.x >> shift); i < n; i += (int64_t)gridDim.x * per) {
        const int64_t id = load_id(ids, wide, i);
        const bool known = id >= 0 && id < rows;
        const T *src = table + (known ? id : 0) * row_stride;
        for (int64_t at = (int64_t)(blockIdx.y << shift) * VEC + lane * VEC; at < dim;
             at += (int64_t)(gridDim.y << shift) * VEC) {
            Row<T> r = nerf::load_piece(src + at, known ? dim - at : 0);
#pragma unroll
            for (int j = 0; j < VEC; ++j) r.v[j] = (T)(known ? (float)r.v[j] * scale : __builtin_nanf(""));
            nerf::store_piece(out + i * dim + at, r, dim - at);
        }
    }
}

// ------------------------------------------------------------------------------------------------ sort
// Stable least-significant-digit radix sort of (key, position), 32 bits each.  Keys are the ids; ids that give no gradient
// take the key `rows`, behind all others.  A digit has at most 9 bits.
//
// One tile is 1024 threads x ITEMS pairs, a wavefront holding 64 consecutive pairs per step, so that the order inside a
// digit is (wavefront, step, lane).  `rank` finds a pair's place among the equal digits before it: the lanes that share
// its digit by one ballot per bit, plus the count its wavefront kept so far.
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / WAVE, MAX_DIGIT_BITS = 9, MAX_BINS = 1 << MAX_DIGIT_BITS;
constexpr int TILE_ITEMS = 4, TILE = SORT_THREADS * TILE_ITEMS;            // several workgroups
constexpr int ONE_ITEMS = 16, ONE_TILE = SORT_THREADS * ONE_ITEMS;         // one workgroup

__device__ __forceinline__ uint32_t sort_key(const void *ids, int wide, int64_t i, int64_t rows, int64_t padding_idx) {
    const int64_t id = load_id(ids, wide, i);
    return (uint32_t)(id >= 0 && id < rows && id != padding_idx ? id : rows);
}

template <int ITEMS>
struct Tile {
    uint32_t key[ITEMS], pos[ITEMS], place[ITEMS];
};

// counts[w][d] <- number of pairs of wavefront w with digit d; place <- number of such pairs before this one
template <int ITEMS>
__device__ __forceinline__ void rank(Tile<ITEMS> &t, int n_tile, int shift, int bits, uint32_t *counts) {
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1), bins = 1 << bits;
    for (int d = threadIdx.x; d < SORT_WAVES * bins; d += SORT_THREADS) counts[d] = 0;
    __syncthreads();
    volatile uint32_t *mine = counts + wave * bins;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const bool live = (wave * ITEMS + k) * WAVE + lane < n_tile;
        const uint32_t digit = (t.key[k] >> shift) & (bins - 1);
        uint64_t same = __ballot(live);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(live && (digit >> b & 1));
            same &= (digit >> b & 1) ? set : ~set;
        }
        if (live) {
            const uint32_t before = mine[digit];
            t.place[k] = before + __popcll(same & ((1ull << lane) - 1));
            // the first of the lanes that share the digit writes; a wavefront's LDS accesses keep their order
            if ((same & ((1ull << lane) - 1)) == 0) mine[digit] = before + __popcll(same);
        }
    }
    __syncthreads();
}

// counts[w][d] <- start of (d, w) in the order (digit, wavefront), given base[d] (the digit's start) or, without one, the
// digits of this tile alone.  totals[d] <- number of pairs with digit d.  scan: SORT_WAVES + 1 words.
__device__ __forceinline__ void digit_starts(uint32_t *counts, int bits, uint32_t *scan, const uint32_t *base, int base_step,
                                             uint32_t *totals, int totals_step) {
    const int bins = 1 << bits, wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
    uint32_t total = 0;
    if ((int)threadIdx.x < bins)
        for (int w = 0; w < SORT_WAVES; ++w) total += counts[w * bins + threadIdx.x];
    uint32_t incl = total;
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const uint32_t up = __shfl_up(incl, d, WAVE);
        if (lane >= d) incl += up;
    }
    if (lane == WAVE - 1) scan[wave] = incl;
    __syncthreads();
    uint32_t start = incl - total;
    for (int w = 0; w < wave; ++w) start += scan[w];
    if ((int)threadIdx.x < bins) {
        if (totals) totals[(int64_t)threadIdx.x * totals_step] = total;
        if (base) start = base[(int64_t)threadIdx.x * base_step];
        for (int w = 0; w < SORT_WAVES; ++w) {
            const uint32_t c = counts[w * bins + threadIdx.x];
            counts[w * bins + threadIdx.x] = start;
            start += c;
        }
    }
    __syncthreads();
}

// All passes in one workgroup: up to ONE_TILE pairs.  The pairs go through LDS between two passes.
__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_one_kernel(const void *__restrict__ ids, int wide, int n,
                                                                          int64_t rows, int64_t padding_idx, int passes,
                                                                          int bits, uint32_t *__restrict__ keys,
                                                                          uint32_t *__restrict__ order) {
    extern __shared__ uint32_t lds[];
    uint32_t *sk = lds, *counts = sk + ONE_TILE, *scan = counts + (SORT_WAVES << bits);
    uint16_t *sp = reinterpret_cast<uint16_t *>(scan + SORT_WAVES);
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
    Tile<ONE_ITEMS> t;
#pragma unroll
    for (int k = 0; k < ONE_ITEMS; ++k) {
        const int i = (wave * ONE_ITEMS + k) * WAVE + lane;
        t.key[k] = i < n ? sort_key(ids, wide, i, rows, padding_idx) : 0;
        t.pos[k] = i;
    }
    for (int p = 0; p < passes; ++p) {
        rank(t, n, p * bits, bits, counts);
        digit_starts(counts, bits, scan, nullptr, 0, nullptr, 0);
#pragma unroll
        for (int k = 0; k < ONE_ITEMS; ++k) {
            const int i = (wave * ONE_ITEMS + k) * WAVE + lane;
            if (i < n) {
                const uint32_t to = counts[(wave << bits) + ((t.key[k] >> (p * bits)) & ((1 << bits) - 1))] + t.place[k];
                sk[to] = t.key[k];
                sp[to] = (uint16_t)t.pos[k];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ONE_ITEMS; ++k) {
            const int i = (wave * ONE_ITEMS + k) * WAVE + lane;
            if (i < n) { t.key[k] = sk[i]; t.pos[k] = sp[i]; }
        }
    }
#pragma unroll
    for (int k = 0; k < ONE_ITEMS; ++k) {
        const int i = (wave * ONE_ITEMS + k) * WAVE + lane;
        if (i < n) { keys[i] = t.key[k]; order[i] = t.pos[k]; }
    }
}

// One pass over many tiles: totals per (digit, tile), their scan, and the move.  `keys_in` null: the first pass reads ids.
__device__ __forceinline__ void load_tile(Tile<TILE_ITEMS> &t, int64_t n, const void *ids, int wide, int64_t rows,
                                          int64_t padding_idx, const uint32_t *keys_in, const uint32_t *order_in) {
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
#pragma unroll
    for (int k = 0; k < TILE_ITEMS; ++k) {
        const int64_t i = (int64_t)blockIdx.x * TILE + (wave * TILE_ITEMS + k) * WAVE + lane;
        t.key[k] = t.pos[k] = 0;
        if (i < n) {
            t.key[k] = keys_in ? keys_in[i] : sort_key(ids, wide, i, rows, padding_idx);
            t.pos[k] = keys_in ? order_in[i] : (uint32_t)i;
        }
    }
}

__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_count_kernel(const void *__restrict__ ids, int wide, int64_t n,
                                                                            int64_t rows, int64_t padding_idx,
                                                                            const uint32_t *__restrict__ keys_in, int shift,
                                                                            int bits, uint32_t *__restrict__ totals) {
    __shared__ uint32_t counts[MAX_BINS];
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS) counts[d] = 0;
    __syncthreads();
    Tile<TILE_ITEMS> t;
    load_tile(t, n, ids, wide, rows, padding_idx, keys_in, keys_in);
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
#pragma unroll
    for (int k = 0; k < TILE_ITEMS; ++k) {
        const int64_t i = (int64_t)blockIdx.x * TILE + (wave * TILE_ITEMS + k) * WAVE + lane;
        if (i < n) atomicAdd(&counts[(t.key[k] >> shift) & (bins - 1)], 1u);   // a count: the order does not matter
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS) totals[(int64_t)d * gridDim.x + blockIdx.x] = counts[d];
}

// totals <- their exclusive prefix sums, one workgroup
__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_scan_kernel(uint32_t *__restrict__ totals, int64_t count) {
    __shared__ uint32_t sums[SORT_WAVES];
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
    const int64_t per = (count + SORT_THREADS - 1) / SORT_THREADS;
    const int64_t lo = per * threadIdx.x < count ? per * threadIdx.x : count, hi = lo + per < count ? lo + per : count;
    uint32_t total = 0;
    for (int64_t i = lo; i < hi; ++i) total += totals[i];
    uint32_t incl = total;
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const uint32_t up = __shfl_up(incl, d, WAVE);
        if (lane >= d) incl += up;
    }
    if (lane == WAVE - 1) sums[wave] = incl;
    __syncthreads();
    uint32_t run = incl - total;
    for (int w = 0; w < wave; ++w) run += sums[w];
    for (int64_t i = lo; i < hi; ++i) {
        const uint32_t c = totals[i];
        totals[i] = run;
        run += c;
    }
}

__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_move_kernel(const void *__restrict__ ids, int wide, int64_t n,
                                                                           int64_t rows, int64_t padding_idx,
                                                                           const uint32_t *__restrict__ keys_in,
                                                                           const uint32_t *__restrict__ order_in, int shift,
                                                                           int bits, const uint32_t *__restrict__ starts,
                                                                           uint32_t *__restrict__ keys,
                                                                           uint32_t *__restrict__ order) {
    __shared__ uint32_t counts[SORT_WAVES * MAX_BINS], scan[SORT_WAVES];
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
    Tile<TILE_ITEMS> t;
    load_tile(t, n, ids, wide, rows, padding_idx, keys_in, order_in);
    const int64_t left = n - (int64_t)blockIdx.x * TILE;
    rank(t, (int)(left < TILE ? left : TILE), shift, bits, counts);
    digit_starts(counts, bits, scan, starts + blockIdx.x, gridDim.x, nullptr, 0);
#pragma unroll
    for (int k = 0; k < TILE_ITEMS; ++k) {
        if ((wave * TILE_ITEMS + k) * WAVE + lane < left) {
            const uint32_t to = counts[(wave << bits) + ((t.key[k] >> shift) & ((1 << bits) - 1))] + t.place[k];
            keys[to] = t.key[k];
            order[to] = t.pos[k];
        }
    }
}

// ------------------------------------------------------------------------------------------------ sums
template <typename T>
__global__ __launch_bounds__(256) void embedding_zero_kernel(T *__restrict__ g_table, int64_t count) {
    Row<T> zero;
#pragma unroll
    for (int j = 0; j < Row<T>::VEC; ++j) zero.v[j] = (T)0.0f;
    for (int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * Row<T>::VEC; at < count;
         at += (int64_t)gridDim.x * 256 * Row<T>::VEC)
        nerf::store_piece(g_table + at, zero, count - at);
}

// partial rows: [chunk][2][dim] fp32 -- 0: the sum of the id that the chunk begins inside of (up to its end, or the whole
// chunk), 1: the sum of the id that begins in the chunk and goes on behind it
template <typename T>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const T *__restrict__ g_out, int64_t n, int64_t dim,
                                                            const uint32_t *__restrict__ keys,
                                                            const uint32_t *__restrict__ order, uint32_t rows, float scale,
                                                            int chunk, int shift, T *__restrict__ g_table,
                                                            float *__restrict__ partial) {
    constexpr int VEC = Row<T>::VEC, AHEAD = 4;
    const int lane = threadIdx.x & ((1 << shift) - 1);
    const int64_t c = (int64_t)blockIdx.x * (256 >> shift) + (threadIdx.x >> shift);
    const int64_t lo = c * chunk, hi = lo + chunk < n ? lo + chunk : n;
    const int64_t at = ((int64_t)(blockIdx.y << shift) + lane) * VEC, left = dim - at;
    if (lo >= n || left <= 0) return;
    uint32_t key = keys[lo];
    bool begins = lo == 0 || keys[lo - 1] != key;
    float sum[VEC] = {};
    auto flush = [&](bool ends) {
        if (key >= rows) return;
        if (begins && ends) {
            Row<T> r;
#pragma unroll
            for (int j = 0; j < VEC; ++j) r.v[j] = (T)(sum[j] * scale);
            nerf::store_piece(g_table + (int64_t)key * dim + at, r, left);
        } else {
            float *dst = partial + (c * 2 + (begins ? 1 : 0)) * dim + at;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (j < left) dst[j] = sum[j];
        }
    };
    for (int64_t i = lo; i < hi; i += AHEAD) {
        uint32_t k[AHEAD];
        Row<T> r[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            k[u] = i + u < hi ? keys[i + u] : rows;
            r[u] = nerf::load_piece(g_out + (int64_t)(k[u] < rows ? order[i + u] : 0) * dim + at, k[u] < rows ? left : 0);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (i + u >= hi) break;
            if (k[u] != key) {
                flush(true);
                key = k[u];
                begins = true;
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum[j] += (float)r[u].v[j];
        }
    }
    flush(hi >= n || keys[hi] != key);
}

// One workgroup per chunk (and 64 columns); it has work only where an id begins in the chunk and goes on behind it.
template <typename T>
__global__ __launch_bounds__(256) void embedding_join_kernel(const uint32_t *__restrict__ keys, int64_t n, int64_t dim,
                                                             uint32_t rows, float scale, int chunk,
                                                             const float *__restrict__ partial, T *__restrict__ g_table) {
    const int64_t c = blockIdx.x, lo = c * chunk, hi = lo + chunk;
    if (hi >= n) return;
    const uint32_t key = keys[hi - 1];
    if (key >= rows || keys[hi] != key) return;
    if (keys[lo] == key && lo > 0 && keys[lo - 1] == key) return;       // it began before
    int64_t a = hi, b = n;                                              // first place behind the id
    while (a < b) {
        const int64_t m = (a + b) >> 1;
        if (keys[m] > key) b = m; else a = m + 1;
    }
    const int64_t last = (a - 1) / chunk;
    __shared__ float part[4][64];
    const int col = threadIdx.x & 63, s = threadIdx.x >> 6;
    const int64_t at = (int64_t)blockIdx.y * 64 + col;
    float sum = 0.0f;
    if (at < dim) {
        if (s == 0) sum = partial[(c * 2 + 1) * dim + at];
        for (int64_t k = c + 1 + s; k <= last; k += 4) sum += partial[k * 2 * dim + at];
    }
    part[s][col] = sum;
    __syncthreads();
    if (s == 0 && at < dim) g_table[(int64_t)key * dim + at] = (T)((part[0][col] + part[1][col] + part[2][col] + part[3][col]) * scale);
}

// ------------------------------------------------------------------------------------------------ plan
struct Plan {
    int bits, passes;                  // of the sort
    int64_t tiles;                     // 0: one workgroup
    int shift;                         // 2^shift lanes per row
    int64_t column_tiles;
    int chunk;                         // sorted pairs per lane group
    int64_t chunks;
    int64_t keys, order, keys2, order2, totals, partial, bytes;   // offsets in the workspace
};

int lane_shift(int64_t pieces) {
    int s = 0;
    while (s < 8 && (1 << s) < pieces) ++s;
    return s;
}

Plan plan_backward(int64_t n, int64_t rows, int64_t dim, int dtype) {
    Plan p;
    int bits = 1;
    while (rows >> bits) ++bits;
    p.passes = (bits + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.tiles = n <= ONE_TILE ? 0 : (n + TILE - 1) / TILE;
    const int64_t pieces = (dim * nerf::dtype_bytes(dtype) + 15) / 16;
    p.shift = lane_shift(pieces);
    p.column_tiles = (pieces + (1 << p.shift) - 1) >> p.shift;
    // about 8 wavefronts per SIMD of the chip, in lane groups; never fewer than 8 pairs a group
    const int64_t groups = ((int64_t)256 * 32 * WAVE >> p.shift) / p.column_tiles;
    int64_t chunk = groups > 0 ? (n + groups - 1) / groups : n;
    if (chunk < 8) chunk = 8;
    p.chunk = (int)chunk;
    p.chunks = (n + chunk - 1) / chunk;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t r = at; at += (bytes + 255) / 256 * 256; return r; };
    p.keys = take(4 * n);
    p.order = take(4 * n);
    const bool twice = p.tiles && p.passes > 1;
    p.keys2 = take(twice ? 4 * n : 0);
    p.order2 = take(twice ? 4 * n : 0);
    p.totals = take(p.tiles ? 4 * (p.tiles << p.bits) : 0);
    p.partial = take(p.chunks * 2 * dim * 4);
    p.bytes = at;
    return p;
}

bool sizes_ok(int64_t n, int64_t rows, int64_t dim) {
    return n >= 0 && n < (int64_t)1 << 31 && rows >= 1 && rows < (int64_t)1 << 31 && dim >= 1 && dim <= (int64_t)1 << 20;
}

template <typename T>
void launch_forward(const void *table, int64_t rows, int64_t row_stride, int64_t dim, const void *ids, int wide, int64_t n,
                    float scale, void *out, hipStream_t stream) {
    const int64_t pieces = (dim + Row<T>::VEC - 1) / Row<T>::VEC;
    const int shift = lane_shift(pieces);
    const int64_t per = 256 >> shift;
    int64_t gx = (n + per - 1) / per, gy = (pieces + (1 << shift) - 1) >> shift;
    if (gx > 256 * 16) gx = 256 * 16;
    if (gy > 64) gy = 64;
    hipLaunchKernelGGL(embedding_kernel<T>, dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, stream,
                       static_cast<const T *>(table), rows, row_stride, dim, ids, wide, n, scale, shift,
                       static_cast<T *>(out));
}

template <typename T>
int launch_backward(const void *g_out, int dtype, int64_t n, int64_t dim, const void *ids, int wide, int64_t rows, float scale,
                    int64_t padding_idx, void *g_table, char *ws, hipStream_t stream) {
    T *gt = static_cast<T *>(g_table);
    const int64_t count = rows * dim;
    int64_t grid = (count + 256 * Row<T>::VEC - 1) / (256 * Row<T>::VEC);
    hipLaunchKernelGGL(embedding_zero_kernel<T>, dim3((unsigned)(grid < 4096 ? grid : 4096)), dim3(256), 0, stream, gt, count);
    if (n == 0) return NERF_OK;
    const Plan p = plan_backward(n, rows, dim, dtype);
    uint32_t *keys = reinterpret_cast<uint32_t *>(ws + p.keys), *order = reinterpret_cast<uint32_t *>(ws + p.order);
    float *partial = reinterpret_cast<float *>(ws + p.partial);
    if (!p.tiles) {
        static nerf::DeviceMask done;
        const int lds = 4 * (ONE_TILE + (SORT_WAVES << p.bits) + SORT_WAVES) + 2 * ONE_TILE;
        if (int rc = nerf::ensure_dynamic_lds(reinterpret_cast<const void *>(embedding_sort_one_kernel), 160 * 1024, done,
                                              "nerf_embedding_backward"))
            return rc;
        hipLaunchKernelGGL(embedding_sort_one_kernel, dim3(1), dim3(SORT_THREADS), lds, stream, ids, wide, (int)n, rows,
                           padding_idx, p.passes, p.bits, keys, order);
    } else {
        uint32_t *totals = reinterpret_cast<uint32_t *>(ws + p.totals);
        // the last pass has to end in `keys`
        uint32_t *k[2] = {keys, reinterpret_cast<uint32_t *>(ws + p.keys2)};
        uint32_t *o[2] = {order, reinterpret_cast<uint32_t *>(ws + p.order2)};
        for (int q = 0; q < p.passes; ++q) {
            const int to = (p.passes - 1 - q) & 1;
            const uint32_t *ki = q ? k[to ^ 1] : nullptr, *oi = q ? o[to ^ 1] : nullptr;
            hipLaunchKernelGGL(embedding_sort_count_kernel, dim3((unsigned)p.tiles), dim3(SORT_THREADS), 0, stream, ids, wide,
                               n, rows, padding_idx, ki, q * p.bits, p.bits, totals);
            hipLaunchKernelGGL(embedding_sort_scan_kernel, dim3(1), dim3(SORT_THREADS), 0, stream, totals, p.tiles << p.bits);
            hipLaunchKernelGGL(embedding_sort_move_kernel, dim3((unsigned)p.tiles), dim3(SORT_THREADS), 0, stream, ids, wide,
                               n, rows, padding_idx, ki, oi, q * p.bits, p.bits, totals, k[to], o[to]);
        }
    }
    const int64_t per = 256 >> p.shift;
    hipLaunchKernelGGL(embedding_sum_kernel<T>, dim3((unsigned)((p.chunks + per - 1) / per), (unsigned)p.column_tiles),
                       dim3(256), 0, stream, static_cast<const T *>(g_out), n, dim, keys, order, (uint32_t)rows, scale,
                       p.chunk, p.shift, gt, partial);
    if (p.chunks > 1)
        hipLaunchKernelGGL(embedding_join_kernel<T>, dim3((unsigned)(p.chunks - 1), (unsigned)((dim + 63) / 64)), dim3(256), 0,
                           stream, keys, n, dim, (uint32_t)rows, scale, p.chunk, partial, gt);
    return NERF_OK;
}

}  // namespace

NERF_API int nerf_embedding(const void *table, int64_t rows, int64_t row_stride, int dtype, int64_t dim, const void *ids,
                            int id_bytes, int64_t n, float scale, void *out, nerf_stream_t stream) {
    NERF_REQUIRE(nerf::known_dtype(dtype), "nerf_embedding: unknown dtype");
    NERF_REQUIRE(id_bytes == 4 || id_bytes == 8, "nerf_embedding: ids are 4 or 8 bytes wide");
    NERF_REQUIRE(sizes_ok(n, rows, dim), "nerf_embedding: size out of range");
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(table && ids && out, "nerf_embedding: null pointer");
    NERF_REQUIRE(rows == 1 || row_stride >= dim, "nerf_embedding: rows overlap (row_stride < dim)");
    NERF_FOR_DTYPE(dtype, T, launch_forward<T>(table, rows, row_stride, dim, ids, id_bytes == 8, n, scale, out,
                                               nerf::as_stream(stream)));
    return nerf::check_launch("nerf_embedding");
}

NERF_API int64_t nerf_embedding_backward_workspace_bytes(int64_t n, int64_t rows, int64_t dim, int dtype) {
    if (!nerf::known_dtype(dtype) || !sizes_ok(n, rows, dim))
        return nerf::fail(NERF_ERR_ARG, "nerf_embedding_backward_workspace_bytes: size out of range"), -1;
    return n ? plan_backward(n, rows, dim, dtype).bytes : 0;
}

NERF_API int nerf_embedding_backward(const void *g_out, int dtype, int64_t n, int64_t dim, const void *ids, int id_bytes,
                                     int64_t rows, float scale, int64_t padding_idx, void *g_table, void *workspace,
                                     nerf_stream_t stream) {
    NERF_REQUIRE(nerf::known_dtype(dtype), "nerf_embedding_backward: unknown dtype");
    NERF_REQUIRE(id_bytes == 4 || id_bytes == 8, "nerf_embedding_backward: ids are 4 or 8 bytes wide");
    NERF_REQUIRE(sizes_ok(n, rows, dim), "nerf_embedding_backward: size out of range");
    NERF_REQUIRE(g_table && (n == 0 || (g_out && ids && workspace)), "nerf_embedding_backward: null pointer");
    int rc = NERF_OK;
    NERF_FOR_DTYPE(dtype, T, rc = launch_backward<T>(g_out, dtype, n, dim, ids, id_bytes == 8, rows, scale, padding_idx,
                                                     g_table, static_cast<char *>(workspace), nerf::as_stream(stream)));
    return rc ? rc : nerf::check_launch("nerf_embedding_backward");
}
