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
template <typename T, bool TINY>
__global__ __launch_bounds__(256) void embedding_kernel(const T *__restrict__ table, int64_t rows, int64_t row_stride,
                                                        int dim, const void *__restrict__ ids, int wide, int64_t n,
                                                        float scale, int shift, T *__restrict__ out) {
    constexpr int VEC = Row<T>::VEC;
    const int per = 256 >> shift, lane = threadIdx.x & ((1 << shift) - 1);
    for (int64_t i = (int64_t)blockIdx.x * per + (threadIdx.x >> shift); i < n; i += (int64_t)gridDim.x * per) {
        const int64_t id = load_id(ids, wide, i);
        const bool known = id >= 0 && id < rows;
        const T *src = table + (known ? id : 0) * row_stride;
        for (int a = (((int)blockIdx.y << shift) + lane) * VEC; a < dim; a += ((int)gridDim.y << shift) * VEC) {
            const nerf::Place<T, TINY> at(a, dim);
            Row<T> r = nerf::load_piece<TINY>(src, at);
#pragma unroll
            for (int j = 0; j < VEC; ++j) r.v[j] = (T)(known ? (float)r.v[j] * scale : __builtin_nanf(""));
            nerf::store_piece<TINY>(out + i * dim, at, r);
        }
    }
}

// ------------------------------------------------------------------------------------------------ zeros
// Rows that no id names are 0, and nobody knows which before the sort: the whole table is cleared, by workgroups that run
// beside the first sorting launch (the clear is the larger part of a large vocabulary's gradient, and the sort keeps few
// CUs busy).  The summing launch comes after both.  A workgroup clears `per` pieces next to each other: 268 MB in 43 us
// (6.2 TB/s); 1024 workgroups striding over the table took 60 us.
template <typename T>
__device__ __forceinline__ void clear(T *g_table, int64_t count, int64_t per, int64_t block) {
    Row<T> zero;
#pragma unroll
    for (int j = 0; j < Row<T>::VEC; ++j) zero.v[j] = (T)0.0f;
    const int64_t whole = count / Row<T>::VEC, hi = (block + 1) * per < whole ? (block + 1) * per : whole;
    for (int64_t i = block * per + threadIdx.x; i < hi; i += blockDim.x) nerf::store_16(g_table + i * Row<T>::VEC, zero);
    if (block == 0 && (int)threadIdx.x < (int)(count - whole * Row<T>::VEC)) g_table[whole * Row<T>::VEC + threadIdx.x] = zero.v[0];
}

template <typename T>
__global__ __launch_bounds__(1024) void embedding_zero_kernel(T *__restrict__ g_table, int64_t count, int64_t per) {
    clear(g_table, count, per, blockIdx.x);
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
constexpr int ONE_TILE = SORT_THREADS * 16;                                // one workgroup, at most

__device__ __forceinline__ uint32_t sort_key(const void *ids, int wide, int64_t i, int64_t rows, int64_t padding_idx) {
    const int64_t id = load_id(ids, wide, i);
    return (uint32_t)(id >= 0 && id < rows && id != padding_idx ? id : rows);
}

// the lanes of `live` whose digit is this lane's
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, uint64_t live) {
    uint32_t lo = (uint32_t)live, hi = (uint32_t)(live >> 32);
    for (int b = 0; b < bits; ++b) {
        const uint32_t mine = (uint32_t)((int32_t)(digit << (31 - b)) >> 31);       // 0 or all ones
        const uint64_t set = __ballot(mine != 0);
        lo &= ~((uint32_t)set ^ mine);
        hi &= ~((uint32_t)(set >> 32) ^ mine);
    }
    return (uint64_t)hi << 32 | lo;
}

template <int ITEMS>
struct Tile {
    uint32_t key[ITEMS], pos[ITEMS], place[ITEMS];
};

// counts[w][d] <- number of pairs of wavefront w with digit d; place <- number of such pairs before this one
template <int ITEMS>
__device__ __forceinline__ void rank(Tile<ITEMS> &t, int n_tile, int shift, int bits, uint32_t *counts) {
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1), bins = 1 << bits;
    const uint64_t below = (1ull << lane) - 1;
    for (int d = threadIdx.x; d < SORT_WAVES * bins; d += SORT_THREADS) counts[d] = 0;
    __syncthreads();
    volatile uint32_t *mine = counts + wave * bins;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int first = (wave * ITEMS + k) * WAVE;
        if (first >= n_tile) break;
        const bool live = first + lane < n_tile;
        const uint32_t digit = (t.key[k] >> shift) & (bins - 1);
        const uint64_t same = same_digit(digit, bits, __ballot(live));
        if (live) {
            const uint32_t before = mine[digit];
            t.place[k] = before + __popcll(same & below);
            // the first of the lanes that share the digit writes; a wavefront's LDS accesses keep their order
            if ((same & below) == 0) mine[digit] = before + __popcll(same);
        }
    }
    __syncthreads();
}

// Exclusive prefix sum of one value per thread.  sums: SORT_WAVES words.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t *sums) {
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
    uint32_t incl = v;
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const uint32_t up = __shfl_up(incl, d, WAVE);
        if (lane >= d) incl += up;
    }
    if (lane == WAVE - 1) sums[wave] = incl;
    __syncthreads();
    uint32_t start = incl - v;
    for (int w = 0; w < wave; ++w) start += sums[w];
    return start;
}

// counts[w][d] <- place of the first pair of wavefront w with digit d.  Of one tile alone (`totals` null), or of tile
// blockIdx.x among many: totals[d] = pairs with digit d in all tiles, before[d] = in the tiles before this one.
__device__ __forceinline__ void digit_starts(uint32_t *counts, int bits, uint32_t *sums, const uint32_t *totals,
                                             const uint32_t *before, int64_t before_step) {
    const int bins = 1 << bits;
    uint32_t total = 0;
    if ((int)threadIdx.x < bins) {
        if (totals)
            total = totals[threadIdx.x];
        else
            for (int w = 0; w < SORT_WAVES; ++w) total += counts[w * bins + threadIdx.x];
    }
    uint32_t start = block_prefix(total, sums);
    if ((int)threadIdx.x < bins) {
        if (totals) start += before[threadIdx.x * before_step];
        for (int w = 0; w < SORT_WAVES; ++w) {
            const uint32_t c = counts[w * bins + threadIdx.x];
            counts[w * bins + threadIdx.x] = start;
            start += c;
        }
    }
    __syncthreads();
}

// All passes in one workgroup (the first; the others clear the table): up to 1024 x ITEMS pairs.  Between two passes the
// pairs go through LDS.
template <int ITEMS>
constexpr int one_lds_bytes(int bits) {
    return 4 * (SORT_THREADS * ITEMS + (SORT_WAVES << bits) + SORT_WAVES) + 2 * SORT_THREADS * ITEMS;
}

template <typename T, int ITEMS>
__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_one_kernel(const void *__restrict__ ids, int wide, int n,
                                                                          int64_t rows, int64_t padding_idx, int passes,
                                                                          int bits, uint32_t *__restrict__ keys,
                                                                          uint32_t *__restrict__ order,
                                                                          T *__restrict__ g_table, int64_t count, int64_t per) {
    if (blockIdx.x > 0) {
        clear(g_table, count, per, blockIdx.x - 1);
        return;
    }
    extern __shared__ uint32_t lds[];
    uint32_t *sk = lds, *counts = sk + SORT_THREADS * ITEMS, *sums = counts + (SORT_WAVES << bits);
    uint16_t *sp = reinterpret_cast<uint16_t *>(sums + SORT_WAVES);
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
    Tile<ITEMS> t;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = (wave * ITEMS + k) * WAVE + lane;
        t.key[k] = i < n ? sort_key(ids, wide, i, rows, padding_idx) : 0;
        t.pos[k] = i;
    }
    for (int p = 0; p < passes; ++p) {
        rank(t, n, p * bits, bits, counts);
        digit_starts(counts, bits, sums, nullptr, nullptr, 0);
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = (wave * ITEMS + k) * WAVE + lane;
            if (i < n) {
                const uint32_t to = counts[(wave << bits) + ((t.key[k] >> (p * bits)) & ((1 << bits) - 1))] + t.place[k];
                sk[to] = t.key[k];
                sp[to] = (uint16_t)t.pos[k];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = (wave * ITEMS + k) * WAVE + lane;
            if (i < n) { t.key[k] = sk[i]; t.pos[k] = sp[i]; }
        }
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = (wave * ITEMS + k) * WAVE + lane;
        if (i < n) { keys[i] = t.key[k]; order[i] = t.pos[k]; }
    }
}

// One pass over many tiles: counts [digit][tile]; their prefix sums along the tiles and the totals of the digits, one
// workgroup a digit; the move.  `keys_in` null: the first pass, which reads the ids (and has workgroups that clear).
__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_scan_kernel(uint32_t *__restrict__ counts, int64_t tiles,
                                                                           uint32_t *__restrict__ totals) {
    __shared__ uint32_t sums[2][SORT_WAVES];
    uint32_t *row = counts + blockIdx.x * tiles, carry = 0;
    int half = 0;
    for (int64_t at = 0; at < tiles; at += SORT_THREADS, half ^= 1) {
        const bool live = at + threadIdx.x < tiles;
        const uint32_t v = live ? row[at + threadIdx.x] : 0;
        const uint32_t start = block_prefix(v, sums[half]);
        if (live) row[at + threadIdx.x] = carry + start;
        for (int w = 0; w < SORT_WAVES; ++w) carry += sums[half][w];
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <typename T>
__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_count_kernel(const void *__restrict__ ids, int wide, int64_t n,
                                                                            int64_t rows, int64_t padding_idx,
                                                                            const uint32_t *__restrict__ keys_in, int shift,
                                                                            int bits, int64_t tiles,
                                                                            uint32_t *__restrict__ counts,
                                                                            T *__restrict__ g_table, int64_t count, int64_t per) {
    if (blockIdx.x >= tiles) {
        clear(g_table, count, per, blockIdx.x - tiles);
        return;
    }
    __shared__ uint32_t mine[MAX_BINS];
    const int bins = 1 << bits, wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS) mine[d] = 0;
    __syncthreads();
    uint32_t key[TILE_ITEMS];
#pragma unroll
    for (int k = 0; k < TILE_ITEMS; ++k) {
        const int64_t i = (int64_t)blockIdx.x * TILE + (wave * TILE_ITEMS + k) * WAVE + lane;
        key[k] = i >= n ? 0 : keys_in ? keys_in[i] : sort_key(ids, wide, i, rows, padding_idx);
    }
#pragma unroll
    for (int k = 0; k < TILE_ITEMS; ++k) {
        const int64_t i = (int64_t)blockIdx.x * TILE + (wave * TILE_ITEMS + k) * WAVE + lane;
        const uint32_t digit = (key[k] >> shift) & (bins - 1);
        const uint64_t same = same_digit(digit, bits, __ballot(i < n));
        // one addition per digit and wavefront; counts: the order does not matter
        if (i < n && (same & ((1ull << lane) - 1)) == 0) atomicAdd(&mine[digit], (uint32_t)__popcll(same));
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += SORT_THREADS) counts[(int64_t)d * tiles + blockIdx.x] = mine[d];
}

__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_move_kernel(const void *__restrict__ ids, int wide, int64_t n,
                                                                           int64_t rows, int64_t padding_idx,
                                                                           const uint32_t *__restrict__ keys_in,
                                                                           const uint32_t *__restrict__ order_in, int shift,
                                                                           int bits, const uint32_t *__restrict__ totals,
                                                                           const uint32_t *__restrict__ before,
                                                                           uint32_t *__restrict__ keys,
                                                                           uint32_t *__restrict__ order) {
    __shared__ uint32_t counts[SORT_WAVES * MAX_BINS], sums[SORT_WAVES];
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
    Tile<TILE_ITEMS> t;
#pragma unroll
    for (int k = 0; k < TILE_ITEMS; ++k) {
        const int64_t i = (int64_t)blockIdx.x * TILE + (wave * TILE_ITEMS + k) * WAVE + lane;
        t.key[k] = t.pos[k] = 0;
        if (i < n) {
            t.key[k] = keys_in ? keys_in[i] : sort_key(ids, wide, i, rows, padding_idx);
            t.pos[k] = keys_in ? order_in[i] : (uint32_t)i;
        }
    }
    const int64_t left = n - (int64_t)blockIdx.x * TILE;
    rank(t, (int)(left < TILE ? left : TILE), shift, bits, counts);
    digit_starts(counts, bits, sums, totals, before + blockIdx.x, gridDim.x);
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
// A workgroup takes a span of the sorted pairs, cut into chunks: 2^shift lanes walk one chunk, a piece of the columns each.
// An id that begins and ends in a chunk is stored by its lanes; what an id leaves in several chunks of the workgroup meets
// in LDS, chunk after chunk.  An id that crosses workgroups leaves partial rows [workgroup][2][dim] (fp32): 0 -- the sum of
// the id that the span begins inside of, 1 -- the sum of the id that begins in the span and goes on behind it, where
// embedding_join_kernel has a row to add up (goes_on).
constexpr int SUM_THREADS = 256;

template <typename T, bool TINY>
__global__ __launch_bounds__(SUM_THREADS) void embedding_sum_kernel(const T *__restrict__ g_out, int64_t n, int dim,
                                                                    const uint32_t *__restrict__ keys,
                                                                    const uint32_t *__restrict__ order, uint32_t rows,
                                                                    float scale, int chunk, int shift,
                                                                    T *__restrict__ g_table, float *__restrict__ partial,
                                                                    uint32_t *__restrict__ goes_on) {
    constexpr int VEC = Row<T>::VEC, AHEAD = 8;
    // what a chunk has for its neighbours: HEAD -- its first id began before it; THROUGH -- and goes on behind it;
    // TAIL -- its last id begins in it and goes on behind it
    constexpr uint32_t HEAD = 1, THROUGH = 2, TAIL = 4;
    __shared__ float part[2][SUM_THREADS * VEC];              // [head, tail][chunk][column]
    __shared__ uint32_t first_key[SUM_THREADS], kind[SUM_THREADS];
    const int group = threadIdx.x >> shift, groups = SUM_THREADS >> shift, lane = threadIdx.x & ((1 << shift) - 1);
    const int width = VEC << shift;
    const int64_t span = (int64_t)blockIdx.x * groups * chunk;
    const int64_t lo = span + (int64_t)group * chunk, hi = lo + chunk < n ? lo + chunk : n;
    const int column = blockIdx.y * width;
    const nerf::Place<T, TINY> at(column + lane * VEC, dim);
    if (lo < n && at.live()) {
        uint32_t k[AHEAD], o[AHEAD];
        auto fetch = [&](int64_t i) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int64_t j = i + u < hi ? i + u : hi - 1;
                k[u] = keys[j];
                o[u] = order[j];
            }
        };
        const uint32_t before = lo > 0 ? keys[lo - 1] : ~0u, behind = hi < n ? keys[hi] : ~0u;
        fetch(lo);
        uint32_t key = k[0], mark = 0;
        bool begins = before != key;
        const uint32_t first = key;
        float sum[VEC] = {};
        auto flush = [&](bool ends) {
            if (key >= rows) return;
            if (begins && ends) {
                Row<T> r;
#pragma unroll
                for (int j = 0; j < VEC; ++j) r.v[j] = (T)(sum[j] * scale);
                nerf::store_piece<TINY>(g_table + (int64_t)key * dim, at, r);
            } else {
                mark |= begins ? TAIL : ends ? HEAD : HEAD | THROUGH;
                float *dst = part[begins ? 1 : 0] + threadIdx.x * VEC - at.skip;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (at.own(j)) dst[j] = sum[j];
            }
        };
        for (int64_t i = lo; i < hi; i += AHEAD) {
            // the rows of this step are on their way while the ids of the next one are read (rows of ids that give no
            // gradient as well: their sum goes nowhere)
            Row<T> r[AHEAD];
            uint32_t now[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                now[u] = k[u];
                r[u] = nerf::load_piece<TINY>(g_out + (int64_t)o[u] * dim, at);
            }
            if (i + AHEAD < hi) fetch(i + AHEAD);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (i + u >= hi) break;
                if (now[u] != key) {
                    flush(true);
                    key = now[u];
                    begins = true;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) sum[j] = 0.0f;
                }
#pragma unroll
                for (int j = 0; j < VEC; ++j) sum[j] += (float)r[u].v[j];
            }
        }
        flush(behind != key);
        if (lane == 0) {
            first_key[group] = first;
            kind[group] = mark;
        }
    }
    __syncthreads();
    // the chunks of this workgroup in order, one thread a column
    for (int c = threadIdx.x; c < width && column + c < dim; c += SUM_THREADS) {
        float sum = 0.0f;
        bool open = false, here = false;                      // an id is open; it began in this workgroup
        for (int g = 0; g < groups && span + (int64_t)g * chunk < n; ++g) {
            const uint32_t mark = kind[g];
            if (mark & HEAD) {                                // the open id goes on
                sum += part[0][g * width + c];
                open = true;
                if (!(mark & THROUGH)) {
                    if (here) g_table[(int64_t)first_key[g] * dim + column + c] = (T)(sum * scale);
                    else partial[(int64_t)blockIdx.x * 2 * dim + column + c] = sum;
                    open = false;
                }
            }
            if (mark & TAIL) {
                sum = part[1][g * width + c];
                open = here = true;
            }
        }
        if (open) partial[((int64_t)blockIdx.x * 2 + (here ? 1 : 0)) * dim + column + c] = sum;
        if (blockIdx.y == 0 && c == 0) goes_on[blockIdx.x] = open && here;
    }
}

// One workgroup a span and 256 columns, 4 a lane; it has work where an id begins in the span and goes on behind it: the
// first partial row and those of the spans that follow, one wavefront every fourth of them.
template <typename T, bool TINY>
__global__ __launch_bounds__(256) void embedding_join_kernel(const uint32_t *__restrict__ keys, int64_t n, int dim,
                                                             float scale, int64_t span, const float *__restrict__ partial,
                                                             const uint32_t *__restrict__ goes_on, T *__restrict__ g_table) {
    __shared__ float part[4][256];
    const int64_t c = blockIdx.x, spans = (n + span - 1) / span;
    if (!goes_on[c]) return;
    const int lane = threadIdx.x & 63, s = threadIdx.x >> 6;
    const uint32_t key = keys[(c + 1) * span];
    // the last span that begins inside of the id: 64 spans a step, the steps growing by 64 while all of them do
    int64_t last = c + 1, step = 1;
    for (bool grow = true; step > 0;) {
        const int64_t probe = last + (lane + 1) * step;
        const uint64_t in = __ballot(probe < spans && keys[probe * span] == key);
        const int more = in == ~0ull ? 64 : __ffsll((long long)~in) - 1;
        last += more * step;
        if (more < 64) grow = false;
        step = grow ? step * 64 : step / 64;
    }
    for (int base = blockIdx.y * 256; base < dim; base += gridDim.y * 256) {
        const nerf::Place<float, TINY> at(base + lane * 4, dim);
        float sum[4] = {};
        auto add = [&](int64_t k, int which) {
            const Row<float> r = nerf::load_piece<TINY>(partial + (k * 2 + which) * dim, at);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] += r.v[j];
        };
        if (s == 0) add(c, 1);
#pragma unroll 4
        for (int64_t k = c + 1 + s; k <= last; k += 4) add(k, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at.own(j)) part[s][at.at + j - base] = sum[j];
        __syncthreads();
        const int col = threadIdx.x;
        if (base + col < dim)
            g_table[(int64_t)key * dim + base + col] = (T)((part[0][col] + part[1][col] + part[2][col] + part[3][col]) * scale);
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ plan
struct Plan {
    int bits, passes;                  // of the sort
    int64_t tiles;                     // 0: one workgroup
    int shift;                         // 2^shift lanes per row
    int64_t column_tiles;
    int chunk;                         // sorted pairs per lane group
    int64_t spans;                     // workgroups of the sum, along the pairs
    int64_t keys, order, keys2, order2, counts, totals, partial, goes_on, bytes;   // offsets in the workspace
};

int lane_shift(int64_t pieces) {
    int s = 0;
    while (s < 8 && (1 << s) < pieces) ++s;
    return s;
}

// Of the sum: at least 8 lanes a row, or the chunks of a workgroup, added one after another, become too many (dim 1, 16384
// pairs: 256 chunks took 37 us).
constexpr int MIN_SUM_SHIFT = 3;

Plan plan_backward(int64_t n, int64_t rows, int64_t dim, int dtype) {
    Plan p;
    int bits = 1;
    while (rows >> bits) ++bits;
    p.passes = (bits + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
    p.bits = (bits + p.passes - 1) / p.passes;
    p.tiles = n <= ONE_TILE ? 0 : (n + TILE - 1) / TILE;
    const int64_t pieces = (dim * nerf::dtype_bytes(dtype) + 15) / 16;
    p.shift = lane_shift(pieces) > MIN_SUM_SHIFT ? lane_shift(pieces) : MIN_SUM_SHIFT;
    p.column_tiles = (pieces + (1 << p.shift) - 1) >> p.shift;
    // about 8 wavefronts per SIMD of the chip, in lane groups; never fewer than 8 pairs a group
    const int64_t groups = ((int64_t)256 * 32 * WAVE >> p.shift) / p.column_tiles;
    int64_t chunk = groups > 0 ? (n + groups - 1) / groups : n;
    if (chunk < 8) chunk = 8;
    p.chunk = (int)chunk;
    const int64_t span = chunk * (SUM_THREADS >> p.shift);
    p.spans = (n + span - 1) / span;
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t r = at; at += (bytes + 255) / 256 * 256; return r; };
    p.keys = take(4 * n);
    p.order = take(4 * n);
    const bool twice = p.tiles && p.passes > 1;
    p.keys2 = take(twice ? 4 * n : 0);
    p.order2 = take(twice ? 4 * n : 0);
    p.counts = take(p.tiles ? 4 * (p.tiles << p.bits) : 0);
    p.totals = take(p.tiles ? 4 << p.bits : 0);
    p.partial = take(p.spans * 2 * dim * 4);
    p.goes_on = take(4 * p.spans);
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
    auto kernel = dim < Row<T>::VEC ? embedding_kernel<T, true> : embedding_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, stream, static_cast<const T *>(table), rows,
                       row_stride, (int)dim, ids, wide, n, scale, shift, static_cast<T *>(out));
}

template <typename T, int ITEMS>
int launch_sort_one(const Plan &p, int64_t clear_blocks, int64_t per, const void *ids, int wide, int64_t n, int64_t rows,
                    int64_t padding_idx, uint32_t *keys, uint32_t *order, T *g_table, int64_t count,
                    hipStream_t stream) {
    static nerf::DeviceMask done;
    auto kernel = embedding_sort_one_kernel<T, ITEMS>;
    if (int rc = nerf::ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), one_lds_bytes<ITEMS>(MAX_DIGIT_BITS), done,
                                          "nerf_embedding_backward"))
        return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(1 + clear_blocks)), dim3(SORT_THREADS), one_lds_bytes<ITEMS>(p.bits), stream,
                       ids, wide, (int)n, rows, padding_idx, p.passes, p.bits, keys, order, g_table, count, per);
    return NERF_OK;
}

template <typename T>
int launch_backward(const void *g_out, int dtype, int64_t n, int64_t dim, const void *ids, int wide, int64_t rows, float scale,
                    int64_t padding_idx, void *g_table, char *ws, hipStream_t stream) {
    T *gt = static_cast<T *>(g_table);
    const int64_t count = rows * dim, pieces = (count + Row<T>::VEC - 1) / Row<T>::VEC;
    int64_t clear_blocks = (pieces + SORT_THREADS - 1) / SORT_THREADS;
    if (clear_blocks > 1024) clear_blocks = 1024;
    const int64_t per = (pieces + clear_blocks - 1) / clear_blocks;
    if (n == 0) {
        hipLaunchKernelGGL(embedding_zero_kernel<T>, dim3((unsigned)clear_blocks), dim3(SORT_THREADS), 0, stream, gt, count, per);
        return NERF_OK;
    }
    const Plan p = plan_backward(n, rows, dim, dtype);
    auto words = [&](int64_t offset) { return reinterpret_cast<uint32_t *>(ws + offset); };
    uint32_t *keys = words(p.keys), *order = words(p.order);
    float *partial = reinterpret_cast<float *>(ws + p.partial);
    if (!p.tiles) {
        auto sort = n <= SORT_THREADS       ? launch_sort_one<T, 1>
                    : n <= SORT_THREADS * 4 ? launch_sort_one<T, 4>
                                            : launch_sort_one<T, 16>;
        if (int rc = sort(p, clear_blocks, per, ids, wide, n, rows, padding_idx, keys, order, gt, count, stream)) return rc;
    } else {
        // the last pass has to end in `keys`
        uint32_t *k[2] = {keys, words(p.keys2)}, *o[2] = {order, words(p.order2)};
        for (int q = 0; q < p.passes; ++q) {
            const int to = (p.passes - 1 - q) & 1;
            const uint32_t *ki = q ? k[to ^ 1] : nullptr, *oi = q ? o[to ^ 1] : nullptr;
            hipLaunchKernelGGL(embedding_sort_count_kernel<T>, dim3((unsigned)(p.tiles + (q ? 0 : clear_blocks))),
                               dim3(SORT_THREADS), 0, stream, ids, wide, n, rows, padding_idx, ki, q * p.bits, p.bits, p.tiles,
                               words(p.counts), gt, count, per);
            hipLaunchKernelGGL(embedding_sort_scan_kernel, dim3(1u << p.bits), dim3(SORT_THREADS), 0, stream, words(p.counts),
                               p.tiles, words(p.totals));
            hipLaunchKernelGGL(embedding_sort_move_kernel, dim3((unsigned)p.tiles), dim3(SORT_THREADS), 0, stream, ids, wide,
                               n, rows, padding_idx, ki, oi, q * p.bits, p.bits, words(p.totals), words(p.counts), k[to], o[to]);
        }
    }
    auto sum = dim < Row<T>::VEC ? embedding_sum_kernel<T, true> : embedding_sum_kernel<T, false>;
    hipLaunchKernelGGL(sum, dim3((unsigned)p.spans, (unsigned)p.column_tiles), dim3(SUM_THREADS), 0, stream,
                       static_cast<const T *>(g_out), n, (int)dim, keys, order, (uint32_t)rows, scale, p.chunk, p.shift, gt, partial,
                       words(p.goes_on));
    if (p.spans > 1) {
        int64_t gy = (dim + 255) / 256;
        auto join = dim < Row<float>::VEC ? embedding_join_kernel<T, true> : embedding_join_kernel<T, false>;
        hipLaunchKernelGGL(join, dim3((unsigned)(p.spans - 1), (unsigned)(gy < 16 ? gy : 16)), dim3(256), 0, stream, keys, n,
                           (int)dim, scale, (int64_t)p.chunk * (SUM_THREADS >> p.shift), partial, words(p.goes_on), gt);
    }
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
