// Embedding lookup with scaling, and its gradient by sorted ids.
//
//   out[i] = scale * table[ids[i]]
//   g_table[v] = scale * sum over { i : ids[i] = v, v != padding_idx } of g_out[i]
//
// An id outside [0, rows) is never used as an address: its output row is NaN, its gradient is dropped.
//
// Gradient: the pairs (id, position) are sorted by id with a stable radix sort, so that the rows of one id stand together
// in the order they came in.  The sorted list is cut into chunks; a lane group walks one chunk with the running sum in
// registers and stores a row of the table when its id ends.  An id that crosses chunks leaves fp32 partial rows: those of one
// workgroup are added in the order of the chunks, those of several by lane groups that take every so many of them each.  No
// atomics on values and an order that follows from the ids and the sizes: the same bits every run.  A table of few rows takes
// a shorter way (embedding_few_kernel).
//
// Lookup: bound by HBM, 16384 rows of 2048 bf16 in 17.5 us; one row in 1.9 us.  Gradient of 16384 x 1024 bf16 into 131072
// rows: 66 us, of which the 268 MB of the table take 43 at the rate of a clear: 11 + 11 us for the sort, which clears 126 MB
// of it meanwhile, 35 for the sums and the rest of the table, 5 to join.  786432 x 48 fp32 into 100 rows: 34 + 6 us, 4.6 TB/s
// in the first.
#include "rows.h"

namespace {

using nerf::Row;

__device__ __forceinline__ int64_t load_id(const void *ids, int wide, int64_t i) {
    return wide ? static_cast<const int64_t *>(ids)[i] : (int64_t) static_cast<const int32_t *>(ids)[i];
}

// Rows of up to 256 pieces stand in a workgroup lane by lane, whatever their length: thread t has piece t % pieces of row
// t / pieces (t < 1024 and pieces <= 256: `magic` = ceil(2^20 / pieces) divides exactly).  Longer rows take a workgroup each,
// STEPS pieces of a lane on their way at once.  Every workgroup takes its rows once, in the order of the output's addresses.
template <typename T, bool TINY, int STEPS>
__global__ __launch_bounds__(1024) void embedding_kernel(const T *__restrict__ table, int64_t rows, int64_t row_stride,
                                                         int dim, const void *__restrict__ ids, int wide, int64_t n,
                                                         float scale, int pieces, uint32_t magic, int per,
                                                         T *__restrict__ out) {
    constexpr int VEC = Row<T>::VEC;
    const int mine = STEPS > 1 ? 0 : (int)(threadIdx.x * magic >> 20), lane = (int)threadIdx.x - mine * pieces;
    const int64_t i = (int64_t)blockIdx.x * per + mine;
    if (i >= n || mine >= per) return;
    const int64_t id = load_id(ids, wide, i);
    const bool known = id >= 0 && id < rows;
    const T *src = table + (known ? id : 0) * row_stride;
    T *dst = out + i * dim;
    const float factor = known ? scale : __builtin_nanf("");
    const int step = blockDim.x * VEC;
    for (int first = lane * VEC; first < dim; first += STEPS * step) {
        Row<T> r[STEPS];
#pragma unroll
        for (int k = 0; k < STEPS; ++k) r[k] = nerf::load_piece<TINY>(src, nerf::Place<T, TINY>(first + k * step, dim));
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) r[k].v[j] = (T)((float)r[k].v[j] * factor);
            nerf::store_piece<TINY>(dst, nerf::Place<T, TINY>(first + k * step, dim), r[k]);
        }
        if (STEPS == 1) break;
    }
}

// ------------------------------------------------------------------------------------------------ zeros
// Rows that no id names are 0.  Clearing a large vocabulary's table is most of its gradient's work, so it goes beside the
// launches that leave the chip idle: workgroups of the first sorting launches clear the first rows whatever the ids are (as
// many as the sort takes time for), and workgroups of the summing launch, which can look rows up in the sorted ids, clear
// those of the others that nothing will be stored to.
//
// A workgroup clears `per` pieces next to each other: 268 MB in 43 us (6.2 TB/s); 1024 workgroups striding over the table
// took 60 us.
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
// take the key `rows`, behind all others.  A digit has at most 10 bits (a thread a digit).
//
// One tile is 1024 threads x ITEMS pairs, a wavefront holding 64 consecutive pairs per step, so that the order inside a
// digit is (wavefront, step, lane).  `rank` finds a pair's place among the equal digits before it: the lanes that share
// its digit by one ballot per bit, plus the count its wavefront kept so far.
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / WAVE, MAX_DIGIT_BITS = 10, MAX_BINS = 1 << MAX_DIGIT_BITS;
constexpr int TILE_ITEMS = 4, TILE = SORT_THREADS * TILE_ITEMS;            // of a pass over many tiles
constexpr int MERGE_TILES = 32, MERGE_MOST = MERGE_TILES * SORT_THREADS;   // sorted tiles of 1024, merged

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
template <int ITEMS, int WAVES = SORT_WAVES>
__device__ __forceinline__ void rank(Tile<ITEMS> &t, int n_tile, int shift, int bits, uint32_t *counts) {
    const int wave = threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1), bins = 1 << bits;
    const uint64_t below = (1ull << lane) - 1;
    for (int d = threadIdx.x; d < WAVES * bins; d += WAVES * WAVE) counts[d] = 0;
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

// Exclusive prefix sum of one value per thread.  sums: a word per wavefront.
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

// Up to MERGE_MOST pairs: every workgroup sorts 1024 of them in LDS, all passes, and one more launch merges.
template <typename T>
__global__ __launch_bounds__(SORT_THREADS) void embedding_sort_tile_kernel(const void *__restrict__ ids, int wide, int n,
                                                                           int64_t rows, int64_t padding_idx, int passes,
                                                                           int bits, int tiles, uint32_t *__restrict__ keys,
                                                                           uint32_t *__restrict__ order,
                                                                           T *__restrict__ g_table, int64_t count, int64_t per) {
    if ((int)blockIdx.x >= tiles) {
        clear(g_table, count, per, blockIdx.x - tiles);
        return;
    }
    __shared__ uint32_t counts[SORT_WAVES * MAX_BINS], sums[SORT_WAVES], sk[SORT_THREADS], sp[SORT_THREADS];
    const int wave = threadIdx.x / WAVE, begin = blockIdx.x * SORT_THREADS, mine = n - begin < SORT_THREADS ? n - begin : SORT_THREADS;
    const int i = threadIdx.x;
    Tile<1> t;
    t.key[0] = i < mine ? sort_key(ids, wide, begin + i, rows, padding_idx) : 0;
    t.pos[0] = begin + i;
    for (int p = 0; p < passes; ++p) {
        rank(t, mine, p * bits, bits, counts);
        digit_starts(counts, bits, sums, nullptr, nullptr, 0);
        if (i < mine) {
            const uint32_t to = counts[(wave << bits) + ((t.key[0] >> (p * bits)) & ((1 << bits) - 1))] + t.place[0];
            sk[to] = t.key[0];
            sp[to] = t.pos[0];
        }
        __syncthreads();
        if (i < mine) { t.key[0] = sk[i]; t.pos[0] = sp[i]; }
    }
    if (i < mine) { keys[begin + i] = t.key[0]; order[begin + i] = t.pos[0]; }
}

// A pair's place among all: its place in its own tile, the pairs of the tiles before that are not larger and those of the
// tiles behind that are smaller.  All keys are in LDS; the searches of a thread do not wait for each other.
template <typename T>
__global__ __launch_bounds__(SORT_THREADS) void embedding_merge_kernel(const uint32_t *__restrict__ keys_in,
                                                                       const uint32_t *__restrict__ order_in, int n, int tiles,
                                                                       uint32_t *__restrict__ keys,
                                                                       uint32_t *__restrict__ order, T *__restrict__ g_table,
                                                                       int64_t count, int64_t per) {
    if ((int)blockIdx.x >= tiles) {
        clear(g_table, count, per, blockIdx.x - tiles);
        return;
    }
    extern __shared__ uint32_t all[];
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
        const int i = t * SORT_THREADS + threadIdx.x;
        const uint32_t k = keys_in[i < n ? i : n - 1];
        all[i] = i < n ? k : ~0u;                            // (nothing: behind all)
    }
    const int own = blockIdx.x, i = own * SORT_THREADS + threadIdx.x;
    const uint32_t pos = i < n ? order_in[i] : 0;
    __syncthreads();
    if (i >= n) return;
    const uint32_t key = all[i];
    uint32_t place = threadIdx.x;
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
        const uint32_t *tile = all + t * SORT_THREADS, limit = key + (t < own ? 1 : 0);      // count the keys below `limit`
        uint32_t below = 0;
#pragma unroll
        for (int step = SORT_THREADS / 2; step > 0; step >>= 1) below += tile[below + step - 1] < limit ? step : 0;
        below += tile[below] < limit ? 1 : 0;
        place += t == own ? 0 : below;
    }
    keys[place] = key;
    order[place] = pos;
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

// first place in keys[lo, hi) that is not below `limit`; a wavefront looks at 64 places a step
__device__ __forceinline__ int64_t wave_lower_bound(const uint32_t *keys, int64_t lo, int64_t hi, uint32_t limit) {
    const int lane = threadIdx.x & (WAVE - 1);
    while (lo < hi) {
        const int64_t step = (hi - lo + WAVE - 1) / WAVE, probe = lo + (lane + 1) * step - 1;
        lo += __popcll(__ballot(probe < hi && keys[probe] < limit)) * step;
        hi = hi < lo + step - 1 ? hi : lo + step - 1;
    }
    return lo;
}

// Clears those of the rows [first, behind) whose id is not in the sorted keys, in the columns of this workgroup.
constexpr int MAX_CLEAR_ROWS = SUM_THREADS;

template <typename T>
__device__ __forceinline__ void clear_absent(T *g_table, int dim, const nerf::Place<T, false> &at, int group, int groups,
                                             const uint32_t *keys, int64_t n, int64_t first, int64_t behind) {
    __shared__ bool present[MAX_CLEAR_ROWS];
    int64_t lo = wave_lower_bound(keys, 0, n, (uint32_t)first), hi = wave_lower_bound(keys, lo, n, (uint32_t)behind);
    const int64_t row = first + threadIdx.x, end = hi;
    if (row < behind) {
        while (lo < hi) {
            const int64_t m = (lo + hi) >> 1;
            if (keys[m] < (uint32_t)row) lo = m + 1; else hi = m;
        }
        present[threadIdx.x] = lo < end && keys[lo] == (uint32_t)row;
    }
    __syncthreads();
    Row<T> zero;
#pragma unroll
    for (int j = 0; j < Row<T>::VEC; ++j) zero.v[j] = (T)0.0f;
    for (int64_t r = first + group; r < behind; r += groups)
        if (!present[r - first]) nerf::store_piece<false>(g_table + r * dim, at, zero);
}

template <typename T, bool TINY>
__global__ __launch_bounds__(SUM_THREADS) void embedding_sum_kernel(const T *__restrict__ g_out, int64_t n, int dim,
                                                                    const uint32_t *__restrict__ keys,
                                                                    const uint32_t *__restrict__ order, uint32_t rows,
                                                                    float scale, int chunk, int shift,
                                                                    T *__restrict__ g_table, float *__restrict__ partial,
                                                                    uint32_t *__restrict__ goes_on, int64_t spans,
                                                                    int64_t cleared, int clear_rows) {
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
    if (!TINY && blockIdx.x >= spans) {                       // beside the sums: rows `cleared` and up, clear_rows each
        const int64_t first = cleared + (blockIdx.x - spans) * clear_rows;
        clear_absent(g_table, dim, nerf::Place<T, false>(at.at + at.skip, dim), group, groups, keys, n, first,
                     first + clear_rows < rows ? first + clear_rows : rows);
        return;
    }
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
        // (sorted: where the first id gives no gradient, none of the chunk does; one at the chunk's end is read for nothing)
        for (int64_t i = first < rows ? lo : hi; i < hi; i += AHEAD) {
            // the rows of this step are on their way while the ids of the next one are read
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

// One workgroup a span and up to 256 columns; it has work where an id begins in the span and goes on behind it: the first
// partial row and those of the spans that follow, 4 columns a lane, 2^shift lanes a row, the lane groups every so many rows
// and then in order.
constexpr int JOIN_THREADS = 256;        // (1024: 15 us more where every second span has work, 16384 x 1024)

template <typename T, bool TINY>
__global__ __launch_bounds__(JOIN_THREADS) void embedding_join_kernel(const uint32_t *__restrict__ keys, int64_t n, int dim,
                                                                      float scale, int64_t span, int shift,
                                                                      const float *__restrict__ partial,
                                                                      const uint32_t *__restrict__ goes_on,
                                                                      T *__restrict__ g_table) {
    __shared__ float part[JOIN_THREADS * 4];
    const int64_t c = blockIdx.x, spans = (n + span - 1) / span;
    if (!goes_on[c]) return;
    const int lane64 = threadIdx.x & (WAVE - 1);
    const uint32_t key = keys[(c + 1) * span];
    // the last span that begins inside of the id: 64 spans a step, the steps growing by 64 while all of them do
    int64_t last = c + 1, step = 1;
    for (bool grow = true; step > 0;) {
        const int64_t probe = last + (lane64 + 1) * step;
        const uint64_t in = __ballot(probe < spans && keys[probe * span] == key);
        const int more = in == ~0ull ? 64 : __ffsll((long long)~in) - 1;
        last += more * step;
        if (more < 64) grow = false;
        step = grow ? step * 64 : step / 64;
    }
    const int group = threadIdx.x >> shift, groups = JOIN_THREADS >> shift, lane = threadIdx.x & ((1 << shift) - 1), width = 4 << shift;
    for (int column = blockIdx.y * width; column < dim; column += gridDim.y * width) {
        const nerf::Place<float, TINY> at(column + lane * 4, dim);
        if (at.live()) {
            float sum[4] = {};
            auto add = [&](int64_t k, int which) {
                const Row<float> r = nerf::load_piece<TINY>(partial + (k * 2 + which) * dim, at);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += r.v[j];
            };
            if (group == 0) add(c, 1);
#pragma unroll 8
            for (int64_t k = c + 1 + group; k <= last; k += groups) add(k, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (at.own(j)) part[group * width + at.at + j - column] = sum[j];
        }
        __syncthreads();
        for (int col = threadIdx.x; col < width && column + col < dim; col += JOIN_THREADS) {
            float s = 0.0f;
            for (int g = 0; g < groups; ++g) s += part[g * width + col];
            g_table[(int64_t)key * dim + column + col] = (T)(s * scale);
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ few rows
// A table of a few rows (codes of views, of token types) that a batch hits again and again: no sort over the batch.  A
// workgroup orders its tile of the batch by id in LDS, sums the runs, and leaves one fp32 partial row per id of the tile,
// [tile][row][dim], and how often each id occurs, [row][tile]; embedding_few_join_kernel adds the partial rows of an id tile
// by tile and stores every row of the table, zeros where there is nothing.  Two launches instead of the two to five of a
// sort: 786432 x 48 fp32 into 100 rows in 42 us instead of 55.
constexpr int FEW_THREADS = 256, FEW_WAVES = FEW_THREADS / WAVE, FEW_ROWS = FEW_THREADS - 1;

template <typename T, bool TINY, int ITEMS>
__global__ __launch_bounds__(FEW_THREADS) void embedding_few_kernel(const T *__restrict__ g_out, int64_t n, int dim,
                                                                    const void *__restrict__ ids, int wide, int rows,
                                                                    int64_t padding_idx, int bits, int shift,
                                                                    float *__restrict__ partial,
                                                                    uint32_t *__restrict__ present) {
    constexpr int VEC = Row<T>::VEC, AHEAD = 8, PAIRS = FEW_THREADS * ITEMS;
    constexpr uint32_t HEAD = 1, THROUGH = 2, TAIL = 4;       // as in embedding_sum_kernel
    __shared__ float part[2][FEW_THREADS * VEC];
    __shared__ uint32_t counts[FEW_WAVES << 8], sums[FEW_WAVES], kind[FEW_THREADS];
    __shared__ uint16_t key_of[PAIRS], place_of[PAIRS], first_key[FEW_THREADS];
    __shared__ int total;
    const int wave = threadIdx.x / WAVE, lane64 = threadIdx.x & (WAVE - 1), tile = blockIdx.x;
    const int64_t base = (int64_t)tile * PAIRS;
    const int mine = n - base < PAIRS ? (int)(n - base) : PAIRS;
    Tile<ITEMS> t;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        t.pos[k] = (wave * ITEMS + k) * WAVE + lane64;
        t.key[k] = (int)t.pos[k] < mine ? sort_key(ids, wide, base + t.pos[k], rows, padding_idx) : 0;
    }
    rank<ITEMS, FEW_WAVES>(t, mine, 0, bits, counts);
    const int bins = 1 << bits, d = threadIdx.x;
    uint32_t c[FEW_WAVES], here = 0;
#pragma unroll
    for (int w = 0; w < FEW_WAVES; ++w) {
        c[w] = d < bins ? counts[w * bins + d] : 0;
        here += c[w];
    }
    uint32_t start = block_prefix(here, sums);
    if (d == rows) total = start;                             // ids that give no gradient stand behind the others
    if (d < rows && blockIdx.y == 0) present[(int64_t)d * gridDim.x + tile] = here;
#pragma unroll
    for (int w = 0; w < FEW_WAVES; ++w) {
        if (d < bins) counts[w * bins + d] = start;
        start += c[w];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        if ((int)t.pos[k] < mine) {
            const uint32_t to = counts[wave * bins + t.key[k]] + t.place[k];
            key_of[to] = (uint16_t)t.key[k];
            place_of[to] = (uint16_t)t.pos[k];
        }
    }
    __syncthreads();
    const int group = threadIdx.x >> shift, groups = FEW_THREADS >> shift, lane = threadIdx.x & ((1 << shift) - 1);
    const int width = VEC << shift, column = blockIdx.y * width, all = total, chunk = (all + groups - 1) / groups;
    const nerf::Place<T, TINY> at(column + lane * VEC, dim);
    const int lo = group * chunk < all ? group * chunk : all, hi = lo + chunk < all ? lo + chunk : all;
    float *out = partial + (int64_t)tile * rows * dim;
    uint32_t mark = 0;
    if (lo < hi && at.live()) {
        uint32_t key = key_of[lo];
        bool begins = lo == 0 || key_of[lo - 1] != key;
        float sum[VEC] = {};
        auto flush = [&](bool ends) {
            if (begins && ends) {
                float *dst = out + (int64_t)key * dim + at.at;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (at.own(j)) dst[j] = sum[j];
            } else {
                mark |= begins ? TAIL : ends ? HEAD : HEAD | THROUGH;
                float *dst = part[begins ? 1 : 0] + threadIdx.x * VEC - at.skip;
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    if (at.own(j)) dst[j] = sum[j];
            }
        };
        if (lane == 0) first_key[group] = (uint16_t)key;
        for (int i = lo; i < hi; i += AHEAD) {
            Row<T> r[AHEAD];
            uint32_t k[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int j = i + u < hi ? i + u : hi - 1;
                k[u] = key_of[j];
                r[u] = nerf::load_piece<TINY>(g_out + (base + place_of[j]) * dim, at);
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
        flush(hi == all || key_of[hi] != key);
    }
    if (lane == 0) kind[group] = mark;
    __syncthreads();
    for (int col = threadIdx.x; col < width && column + col < dim; col += FEW_THREADS) {
        float sum = 0.0f;
        uint32_t open = 0;                                    // the id that `sum` is of
        for (int g = 0; g < groups; ++g) {
            const uint32_t m = kind[g];
            if (m & HEAD) {
                sum += part[0][g * width + col];
                open = first_key[g];
                if (!(m & THROUGH)) out[(int64_t)open * dim + column + col] = sum;
            }
            if (m & TAIL) sum = part[1][g * width + col];
        }
    }
}

// A workgroup adds up 32 columns of a row: the tiles that have it, in order, as a list in LDS, then 8 lanes a partial row,
// every 32nd of them each, then the 32 sums in order.  (Looking each tile up when its turn comes took 20 us instead of 5 for
// 768 tiles.)
template <typename T, bool TINY>
__global__ __launch_bounds__(256) void embedding_few_join_kernel(const float *__restrict__ partial,
                                                                 const uint32_t *__restrict__ present, int64_t tiles, int rows,
                                                                 int dim, float scale, T *__restrict__ g_table) {
    constexpr int GROUPS = 32, WIDTH = 32;
    __shared__ float part[GROUPS * WIDTH];
    __shared__ uint32_t list[256], sums[4];
    const int group = threadIdx.x >> 3, lane = threadIdx.x & 7, row = blockIdx.x, column = blockIdx.y * WIDTH;
    const nerf::Place<float, TINY> at(column + lane * 4, dim);
    float sum[4] = {};
    for (int64_t first = 0; first < tiles; first += 256) {
        const int64_t mine = first + threadIdx.x;
        const bool here = mine < tiles && present[row * tiles + mine] != 0;
        const uint32_t place = block_prefix(here ? 1 : 0, sums);
        if (here) list[place] = (uint32_t)threadIdx.x;
        __syncthreads();
        const int count = sums[0] + sums[1] + sums[2] + sums[3];
        if (at.live()) {
#pragma unroll 4
            for (int k = group; k < count; k += GROUPS) {
                const Row<float> r = nerf::load_piece<TINY>(partial + ((first + list[k]) * rows + row) * dim, at);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += r.v[j];
            }
        }
        __syncthreads();
    }
    if (at.live()) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (at.own(j)) part[group * WIDTH + at.at + j - column] = sum[j];
    }
    __syncthreads();
    if (threadIdx.x < WIDTH && column + (int)threadIdx.x < dim) {
        float s = 0.0f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) s += part[g * WIDTH + threadIdx.x];
        g_table[(int64_t)row * dim + column + threadIdx.x] = (T)(s * scale);
    }
}

// ------------------------------------------------------------------------------------------------ plan
struct Plan {
    bool few;                          // embedding_few_kernel: tiles of few_items * FEW_THREADS, no sort
    int few_items;
    int bits, passes;                  // of the sort
    bool merge;                        // sorted tiles of 1024, merged; otherwise passes over many tiles
    int64_t tiles;
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
    Plan p = {};
    int bits = 1;
    while (rows >> bits) ++bits;
    p.passes = (bits + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
    p.bits = (bits + p.passes - 1) / p.passes;
    const int64_t pieces = (dim * nerf::dtype_bytes(dtype) + 15) / 16;
    p.shift = lane_shift(pieces) > MIN_SUM_SHIFT ? lane_shift(pieces) : MIN_SUM_SHIFT;
    p.column_tiles = (pieces + (1 << p.shift) - 1) >> p.shift;
    p.merge = n <= MERGE_MOST;
    // few: what the tiles leave and the join reads, if every id is in every tile, stays a quarter of the batch -- or 8 MB,
    // where a launch costs more
    p.few_items = n <= 256 * FEW_THREADS ? 1 : 4;
    const int64_t pairs = FEW_THREADS * p.few_items, few_tiles = (n + pairs - 1) / pairs;
    const double left = 2.0 * few_tiles * (rows < pairs ? rows : pairs) * dim * 4, batch = (double)n * dim * nerf::dtype_bytes(dtype);
    p.few = rows <= FEW_ROWS && left <= (batch / 4 > 8e6 ? batch / 4 : 8e6);
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t r = at; at += (bytes + 255) / 256 * 256; return r; };
    if (p.few) {
        p.tiles = few_tiles;
        // a small batch of long rows: fewer lanes a row, so that more workgroups share the columns
        while (p.shift > MIN_SUM_SHIFT && p.tiles * p.column_tiles < 512) {
            --p.shift;
            p.column_tiles = (pieces + (1 << p.shift) - 1) >> p.shift;
        }
        p.counts = take(4 * p.tiles * rows);
        p.partial = take(4 * p.tiles * rows * dim);
        p.bytes = at;
        return p;
    }
    p.tiles = p.merge ? (n + SORT_THREADS - 1) / SORT_THREADS : (n + TILE - 1) / TILE;
    // about 8 wavefronts per SIMD of the chip, in lane groups; never fewer than 8 pairs a group
    const int64_t groups = ((int64_t)256 * 32 * WAVE >> p.shift) / p.column_tiles;
    int64_t chunk = groups > 0 ? (n + groups - 1) / groups : n;
    if (chunk < 8) chunk = 8;
    p.chunk = (int)chunk;
    const int64_t span = chunk * (SUM_THREADS >> p.shift);
    p.spans = (n + span - 1) / span;
    p.keys = take(4 * n);
    p.order = take(4 * n);
    const bool twice = p.merge ? p.tiles > 1 : p.passes > 1;
    p.keys2 = take(twice ? 4 * n : 0);
    p.order2 = take(twice ? 4 * n : 0);
    p.counts = take(p.merge ? 0 : 4 * (p.tiles << p.bits));
    p.totals = take(p.merge ? 0 : 4 << p.bits);
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
    const bool packed = pieces <= 256;
    const int64_t per = packed ? 1024 / pieces : 1;
    const unsigned threads = packed ? (unsigned)((per * pieces + WAVE - 1) / WAVE * WAVE) : 256;
    auto kernel = dim < Row<T>::VEC ? embedding_kernel<T, true, 1> : packed ? embedding_kernel<T, false, 1> : embedding_kernel<T, false, 4>;
    const int64_t most = ((int64_t)1 << 31) / threads * per;                // rows of a launch, whose threads are counted in 32 bits
    for (int64_t at = 0; at < n; at += most) {
        const int64_t count = n - at < most ? n - at : most;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((count + per - 1) / per)), dim3(threads), 0, stream,
                           static_cast<const T *>(table), rows, row_stride, (int)dim,
                           static_cast<const char *>(ids) + at * (wide ? 8 : 4), wide, count, scale, (int)pieces,
                           (uint32_t)(((1 << 20) + pieces - 1) / pieces), (int)per, static_cast<T *>(out) + at * dim);
    }
}

// Unconditional clearing of `count` values, shared out to workgroups of SORT_THREADS.
template <typename T>
struct Clear {
    T *at;
    int64_t count, per, blocks;
    Clear(T *at_, int64_t count_) : at(at_), count(count_) {
        const int64_t pieces = (count + Row<T>::VEC - 1) / Row<T>::VEC;
        blocks = (pieces + SORT_THREADS - 1) / SORT_THREADS;
        if (blocks > 1024) blocks = 1024;
        per = blocks ? (pieces + blocks - 1) / blocks : 0;
    }
};

// What the chip clears while a sorting launch of some 10 us lasts (16384 x 1024 bf16 into 131072 rows: 65 us; 70 with 40 MB, 80
// with none), and the shortest row that the summing launch clears (one of fewer than 32 pieces is stored sooner than looked up).
constexpr int64_t CLEAR_BESIDE_SORT = (int64_t)60 << 20, CLEAR_ABSENT_BYTES = 512;

template <typename T>
int launch_backward(const void *g_out, int dtype, int64_t n, int64_t dim, const void *ids, int wide, int64_t rows, float scale,
                    int64_t padding_idx, void *g_table, char *ws, hipStream_t stream) {
    T *gt = static_cast<T *>(g_table);
    if (n == 0) {
        const Clear<T> all(gt, rows * dim);
        hipLaunchKernelGGL(embedding_zero_kernel<T>, dim3((unsigned)all.blocks), dim3(SORT_THREADS), 0, stream, gt, all.count,
                           all.per);
        return NERF_OK;
    }
    const Plan p = plan_backward(n, rows, dim, dtype);
    auto words = [&](int64_t offset) { return reinterpret_cast<uint32_t *>(ws + offset); };
    uint32_t *keys = words(p.keys), *order = words(p.order);
    float *partial = reinterpret_cast<float *>(ws + p.partial);
    if (p.few) {
        const bool tiny = dim < Row<T>::VEC;
        auto few = p.few_items == 1 ? (tiny ? embedding_few_kernel<T, true, 1> : embedding_few_kernel<T, false, 1>)
                                    : (tiny ? embedding_few_kernel<T, true, 4> : embedding_few_kernel<T, false, 4>);
        hipLaunchKernelGGL(few, dim3((unsigned)p.tiles, (unsigned)p.column_tiles), dim3(FEW_THREADS), 0, stream,
                           static_cast<const T *>(g_out), n, (int)dim, ids, wide, (int)rows, padding_idx, p.bits, p.shift,
                           partial, words(p.counts));
        auto join = dim < Row<float>::VEC ? embedding_few_join_kernel<T, true> : embedding_few_join_kernel<T, false>;
        hipLaunchKernelGGL(join, dim3((unsigned)rows, (unsigned)((dim + 31) / 32)), dim3(256), 0, stream, partial,
                           words(p.counts), p.tiles, (int)rows, (int)dim, scale, gt);
        return NERF_OK;
    }
    // rows cleared beside the first and the second launch of the sort; the summing launch has the others
    const int64_t row_bytes = dim * (int64_t)sizeof(T), beside = CLEAR_BESIDE_SORT / row_bytes;
    const bool second = p.merge && p.tiles > 1;
    const int64_t first_rows = row_bytes < CLEAR_ABSENT_BYTES ? rows : beside < rows ? beside : rows;
    const int64_t cleared = second && first_rows + beside < rows ? first_rows + beside : second ? rows : first_rows;
    const Clear<T> one(gt, first_rows * dim), two(gt + first_rows * dim, (cleared - first_rows) * dim);
    uint32_t *k[2] = {keys, words(p.keys2)}, *o[2] = {order, words(p.order2)};
    if (p.merge) {
        hipLaunchKernelGGL(embedding_sort_tile_kernel<T>, dim3((unsigned)(p.tiles + one.blocks)), dim3(SORT_THREADS), 0, stream,
                           ids, wide, (int)n, rows, padding_idx, p.passes, p.bits, (int)p.tiles, k[second], o[second], one.at,
                           one.count, one.per);
        if (second) {
            static nerf::DeviceMask done;
            auto kernel = embedding_merge_kernel<T>;
            if (int rc = nerf::ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), 4 * MERGE_MOST, done,
                                                  "nerf_embedding_backward"))
                return rc;
            hipLaunchKernelGGL(kernel, dim3((unsigned)(p.tiles + two.blocks)), dim3(SORT_THREADS), 4 * SORT_THREADS * p.tiles,
                               stream, k[1], o[1], (int)n, (int)p.tiles, keys, order, two.at, two.count, two.per);
        }
    } else {
        // the last pass has to end in `keys`
        for (int q = 0; q < p.passes; ++q) {
            const int to = (p.passes - 1 - q) & 1;
            const uint32_t *ki = q ? k[to ^ 1] : nullptr, *oi = q ? o[to ^ 1] : nullptr;
            hipLaunchKernelGGL(embedding_sort_count_kernel<T>, dim3((unsigned)(p.tiles + (q ? 0 : one.blocks))),
                               dim3(SORT_THREADS), 0, stream, ids, wide, n, rows, padding_idx, ki, q * p.bits, p.bits, p.tiles,
                               words(p.counts), one.at, one.count, one.per);
            hipLaunchKernelGGL(embedding_sort_scan_kernel, dim3(1u << p.bits), dim3(SORT_THREADS), 0, stream, words(p.counts),
                               p.tiles, words(p.totals));
            hipLaunchKernelGGL(embedding_sort_move_kernel, dim3((unsigned)p.tiles), dim3(SORT_THREADS), 0, stream, ids, wide,
                               n, rows, padding_idx, ki, oi, q * p.bits, p.bits, words(p.totals), words(p.counts), k[to], o[to]);
        }
    }
    int64_t clear_rows = (128 << 10) / row_bytes;
    clear_rows = clear_rows < 1 ? 1 : clear_rows > MAX_CLEAR_ROWS ? MAX_CLEAR_ROWS : clear_rows;
    const int64_t clear_blocks = (rows - cleared + clear_rows - 1) / clear_rows;
    auto sum = dim < Row<T>::VEC ? embedding_sum_kernel<T, true> : embedding_sum_kernel<T, false>;
    hipLaunchKernelGGL(sum, dim3((unsigned)(p.spans + clear_blocks), (unsigned)p.column_tiles), dim3(SUM_THREADS), 0, stream,
                       static_cast<const T *>(g_out), n, (int)dim, keys, order, (uint32_t)rows, scale, p.chunk, p.shift, gt,
                       partial, words(p.goes_on), p.spans, cleared, (int)clear_rows);
    if (p.spans > 1) {
        const int shift = lane_shift((dim + 3) / 4) < 6 ? lane_shift((dim + 3) / 4) : 6;
        const int64_t gy = (dim + 255) / 256;
        auto join = dim < Row<float>::VEC ? embedding_join_kernel<T, true> : embedding_join_kernel<T, false>;
        hipLaunchKernelGGL(join, dim3((unsigned)(p.spans - 1), (unsigned)(gy < 16 ? gy : 16)), dim3(JOIN_THREADS), 0, stream,
                           keys, n, (int)dim, scale, (int64_t)p.chunk * (SUM_THREADS >> p.shift), shift, partial,
                           words(p.goes_on), gt);
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
