// Rows of a table by index, scaled, and the table's gradient.
//
//   out[i, :] = scale table[idx[i], :]                  an index outside [0, rows) gives a zero row
//   gradient[v, :] = scale sum over idx[i] = v of g[i, :]  in 32 bits; not for such indices, nor for the padding row
//
// The gradient sorts the indices (stable, least significant digit first), so that a row's sum is over a contiguous run of
// the sorted list, in an order that the data alone gives: results are the same from call to call, without atomics on
// floats. Runs are uneven (a common code is met by a large part of all primitives, most rows of a large table by none) and
// the zero rows have to be written too, so the work is cut by the merged list of both (tables of few rows are summed otherwise, see
// small tables below): entry e of row k stands at
// position e + k, behind e entries and the ends of k rows, and the end of a row is an item of its own, which writes
// it. Every group of lanes takes the same number of items whatever the runs are; a sum that crosses groups is carried by a
// segmented scan within the block, and a row that crosses blocks is put together by a second kernel from the blocks' first
// and last pieces, in their order.
#include <algorithm>
#include <type_traits>

#include "internal.h"

namespace efgs {

namespace {

// A lane's part of a row: 16 bytes at any of its type's alignments, or one value where rows are shorter than that. A row's last
// lane takes its last 16 bytes, whatever of them the lane before it has too (both make the same values), so that no access
// stands in a branch: a kernel whose loads are in branches waits for each before it sends the next.
template <typename T, int W> struct Part { typedef T type __attribute__((ext_vector_type(W), aligned(sizeof(T)))); };
template <typename T> struct Part<T, 1> { using type = T; };

template <typename T, int W>
__device__ __forceinline__ typename Part<T, W>::type load_part(const T* p) { return *reinterpret_cast<const typename Part<T, W>::type*>(p); }

template <typename T, int W>
__device__ __forceinline__ float value_of(const typename Part<T, W>::type& v, int k) {
    if constexpr (W == 1) return static_cast<float>(v);
    else return static_cast<float>(v[k]);
}

// a float32 product, then rounded to T: the compiler would make one instruction of both for float16 (v_fma_mixlo_f16), whose
// one rounding now and then gives another value than the multiplication and the cast of a tensor
template <typename T>
__device__ __forceinline__ T scaled(float x, float scale) {
    float y = x * scale;
    asm("" : "+v"(y));
    return static_cast<T>(y);
}

// STREAM: past the caches, for outputs of 96 MB and more. What reads an output next is slower then, more so than the store was
// faster for smaller ones (lookup and a product of it, us, in the caches and past them: 64 MB 45.9 and 47.8, 128 MB 94.5 and 92.3, 576 MB 365 and 353;
// table gradient of 102 MB and a product of it 84.4 and 81.1).
constexpr uint64_t stream_from = 96ull << 20;

template <typename T, int W, bool STREAM>
__device__ __forceinline__ void store_part(T* p, const float* x, float scale) {
    if constexpr (W == 1) {
        *p = scaled<T>(x[0], scale);
    } else {
        typename Part<T, W>::type v;
#pragma unroll
        for (int k = 0; k < W; k++) v[k] = scaled<T>(x[k], scale);
        if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<typename Part<T, W>::type*>(p));
        else *reinterpret_cast<typename Part<T, W>::type*>(p) = v;
    }
}

constexpr uint32_t max_blocks = 1u << 23;  // of a launch of 256 threads (32 bits of threads)

// row of an index, or `rows` for none
__device__ __forceinline__ uint32_t row_of(int64_t index, uint32_t rows) {
    return static_cast<uint64_t>(index) < rows ? static_cast<uint32_t>(index) : rows;
}

// ---- lookup ----------------------------------------------------------------------------------------------------------

constexpr uint32_t lookup_block = 256, lookup_items = 4, lookup_tile = lookup_block * lookup_items;

struct LookupArgs {
    const void* indices;
    const void* table;
    void* out;
    uint64_t row_stride;      // of the table
    uint32_t first, n, rows, columns;  // this launch: indices from `first` on
    uint32_t row_lanes;       // lanes of a row
    uint32_t lanes;           // of them in a block's tile of columns (<= lookup_tile)
    uint32_t lanes_rcp;       // 2^20 / lanes + 1: t / lanes = t * lanes_rcp >> 20 for t < 1024
    uint32_t rows_per_block;
    float scale;
};

// A block takes whole rows (or, past 1,024 lanes, 1,024 lanes of one row), consecutive lanes of it a row's consecutive parts, four
// of them to a thread: four indices, then four parts, then the stores. One, two and four differed little (1M
// rows of 48 floats 59, 58 and 58 us, 16k of 1,024 bfloat16 11.1, 11.7 and 10.6). 4 rows of 4,096 bfloat16 take 3 us, 1M of 8 floats
// 11, 16k of 1,024 bfloat16 12; 1M of 48 floats, 200 MB stored past the caches, 34.
template <typename T, int W, bool STREAM, typename I>
__global__ __launch_bounds__(lookup_block) void embedding_lookup_kernel(LookupArgs a) {
    const uint32_t first_lane = blockIdx.y * lookup_tile, items = a.rows_per_block * a.lanes;
    const uint64_t first_row = a.first + static_cast<uint64_t>(blockIdx.x) * a.rows_per_block;
    uint64_t i[lookup_items];
    uint32_t column[lookup_items], row[lookup_items];
    bool valid[lookup_items];
    typename Part<T, W>::type v[lookup_items];
#pragma unroll
    for (uint32_t k = 0; k < lookup_items; k++) {
        const uint32_t t = k * lookup_block + threadIdx.x, u = min(t, items - 1);
        const uint32_t q = (u * a.lanes_rcp) >> 20, lane = first_lane + u - q * a.lanes;
        valid[k] = t < items && first_row + q < a.n && lane < a.row_lanes;
        i[k] = min(first_row + q, static_cast<uint64_t>(a.n - 1));
        column[k] = min(lane * W, a.columns - W);
        row[k] = row_of(static_cast<const I*>(a.indices)[i[k]], a.rows);
    }
    const uint32_t last_row = a.rows - 1;
#pragma unroll
    for (uint32_t k = 0; k < lookup_items; k++)
        v[k] = load_part<T, W>(static_cast<const T*>(a.table) + min(row[k], last_row) * a.row_stride + column[k]);
#pragma unroll
    for (uint32_t k = 0; k < lookup_items; k++) {
        float x[W];
#pragma unroll
        for (int j = 0; j < W; j++) x[j] = row[k] < a.rows ? value_of<T, W>(v[k], j) : 0.0f;
        if (valid[k]) store_part<T, W, STREAM>(static_cast<T*>(a.out) + i[k] * a.columns + column[k], x, a.scale);
    }
}

// a table without rows
template <typename T>
__global__ __launch_bounds__(lookup_block) void embedding_zero_kernel(T* out, uint64_t n) {
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * lookup_block + threadIdx.x; i < n; i += static_cast<uint64_t>(gridDim.x) * lookup_block)
        out[i] = static_cast<T>(0.0f);
}

// ---- sort --------------------------------------------------------------------------------------------------------------
// Keys are rows (or `rows` for an index that counts nowhere), values the positions of their indices. A pass orders by up
// to 9 bits: every block knows its digits' places (behind all smaller digits, and behind the same digits of earlier blocks)
// and writes its keys there, each at its rank among the equal digits before it. The counts come from a table that a kernel
// of the same blocks writes, or, up to 16,384 keys, from the block's own count of the whole list, which spares that launch (12k
// indices into 50,000 rows of 8 floats 26.3 -> 24.7 us; 20k 25.7 with the table and 27.6 without). Up to 8,192 keys one kernel counts for
// each key the smaller ones (8,000 keys 22, 8,300 in two passes 24).

constexpr uint32_t sort_block = 1024, sort_waves = sort_block / 64;
constexpr uint32_t sort_steps_most = 4;            // keys of a thread in a tile: these, or one
constexpr uint32_t sort_max_blocks = 256, sort_least_bits = 6, sort_most_bits = 9, sort_most_digits = 1u << sort_most_bits;
constexpr uint32_t sort_alone = 16384;              // largest list that every block counts by itself
constexpr uint32_t rank_most = 8192, rank_keys = 16;  // largest list ordered by ranks, and keys of a block

struct SortPass {
    const void* indices;       // first pass: int32 or int64
    const uint2* in;           // later ones: key, value
    uint2* out;
    uint32_t* table;           // blocks x digits
    uint32_t n, rows, padding; // padding: a row that counts nowhere (>= rows: none)
    uint32_t shift, digit_bits;
    uint32_t tiles_per_block;
    uint32_t steps;            // keys of a thread in a tile
};

// I: the indices' type, or uint2 for a later pass
template <typename I>
__device__ __forceinline__ uint32_t key_at(const SortPass& a, uint32_t i) {
    if constexpr (std::is_same_v<I, uint2>) return a.in[i].x;
    else {
        const uint32_t row = row_of(static_cast<const I*>(a.indices)[i], a.rows);
        return row == a.padding ? a.rows : row;
    }
}

__device__ __forceinline__ uint32_t digit_of(const SortPass& a, uint32_t key) { return (key >> a.shift) & ((1u << a.digit_bits) - 1u); }

template <typename I, uint32_t sort_steps>
__global__ __launch_bounds__(sort_block) void sort_count_kernel(SortPass a) {
    constexpr uint32_t sort_tile = sort_block * sort_steps;
    __shared__ uint32_t counts[sort_most_digits];
    const uint32_t digits = 1u << a.digit_bits;
    if (threadIdx.x < digits) counts[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t tile = 0; tile < a.tiles_per_block; tile++) {
        const uint64_t first = (static_cast<uint64_t>(blockIdx.x) * a.tiles_per_block + tile) * sort_tile + threadIdx.x;
        uint32_t key[sort_steps];
#pragma unroll
        for (uint32_t s = 0; s < sort_steps; s++) {
            const uint64_t i = first + s * sort_block;
            key[s] = key_at<I>(a, static_cast<uint32_t>(min(i, static_cast<uint64_t>(a.n - 1))));
        }
#pragma unroll
        for (uint32_t s = 0; s < sort_steps; s++)
            if (first + s * sort_block < a.n) atomicAdd(&counts[digit_of(a, key[s])], 1u);
    }
    __syncthreads();
    if (threadIdx.x < digits) a.table[blockIdx.x * digits + threadIdx.x] = counts[threadIdx.x];
}

template <typename I>
__device__ __forceinline__ uint2 pair_at(const SortPass& a, uint32_t i) {
    if constexpr (std::is_same_v<I, uint2>) return a.in[i];
    else return make_uint2(key_at<I>(a, i), i);
}

// exclusive prefix over the wave's lanes; the wave's total goes to totals[wave]
__device__ __forceinline__ uint32_t wave_exclusive(uint32_t v, uint32_t* totals) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t inclusive = v;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint32_t t = __shfl_up(inclusive, o);
        if (lane >= o) inclusive += t;
    }
    if (lane == 63) totals[threadIdx.x >> 6] = inclusive;
    return inclusive - v;
}

__device__ __forceinline__ uint32_t totals_before(uint32_t wave, const uint32_t* totals) {
    uint32_t sum = 0;
#pragma unroll
    for (uint32_t w = 0; w < sort_most_digits / 64; w++)
        if (w < wave) sum += totals[w];
    return sum;
}

// ALONE: the block counts the digits of the whole list. A tile is put in order in LDS and written from there, so that a wave's
// stores meet few lines (written from the keys' own lanes, a pass over 1M keys took 22 us; 11 now, the count
// 3.5). 16k keys take 9: the chain of ranks, table reads and prefixes bounds it more than the length does.
template <typename I, bool ALONE, uint32_t sort_steps>
__global__ __launch_bounds__(sort_block) void sort_scatter_kernel(SortPass a) {
    constexpr uint32_t sort_tile = sort_block * sort_steps;
    __shared__ uint16_t counts[sort_waves][sort_most_digits];  // keys of each digit in a wave's part of the tile, then their first place in it
    __shared__ uint32_t wave_totals[sort_waves], to_global[sort_most_digits];
    __shared__ uint2 ordered[sort_tile];
    uint32_t* const all = reinterpret_cast<uint32_t*>(ordered);  // before the tiles: keys of each digit, in parts of the list
    uint32_t* const earlier_blocks = all + sort_block;           // and those of them in blocks before this one
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t digits = 1u << a.digit_bits, parts = sort_block >> a.digit_bits;
    const uint64_t begin = static_cast<uint64_t>(blockIdx.x) * a.tiles_per_block * sort_tile;
    if constexpr (ALONE) {
        all[threadIdx.x] = 0;
        __syncthreads();
        constexpr uint32_t at_once = 16;
        const uint32_t part = threadIdx.x & ~(digits - 1u);
        for (uint32_t from = threadIdx.x; from < a.n; from += at_once * sort_block) {
            uint32_t key[at_once];
#pragma unroll
            for (uint32_t s = 0; s < at_once; s++) key[s] = key_at<I>(a, min(from + s * sort_block, a.n - 1));
#pragma unroll
            for (uint32_t s = 0; s < at_once; s++) {
                const uint32_t i = from + s * sort_block, at = part + digit_of(a, key[s]);
                if (i < a.n) atomicAdd(&all[at], i < begin ? 0x10001u : 1u);  // (both counts, 16 bits each)
            }
        }
    } else {
        const uint32_t digit = threadIdx.x & (digits - 1u), part = threadIdx.x >> a.digit_bits, rows = (gridDim.x + parts - 1) / parts;
        uint32_t before = 0, total = 0;
        constexpr uint32_t at_once = 16;
        for (uint32_t k = 0; k < rows; k += at_once) {
            uint32_t c[at_once];
#pragma unroll
            for (uint32_t j = 0; j < at_once; j++) c[j] = a.table[min(part * rows + k + j, gridDim.x - 1) * digits + digit];
#pragma unroll
            for (uint32_t j = 0; j < at_once; j++) {
                const uint32_t b = part * rows + k + j;
                if (k + j >= rows || b >= gridDim.x) c[j] = 0;
                total += c[j];
                before += b < blockIdx.x ? c[j] : 0u;
            }
        }
        all[threadIdx.x] = total;
        earlier_blocks[threadIdx.x] = before;
    }
    __syncthreads();
    const bool owner = threadIdx.x < digits;  // of a digit (whole waves)
    uint32_t place = 0;                       // of its next key
    if (owner) {
        uint32_t before = 0, total = 0;
        for (uint32_t p = 0; p < parts; p++) {
            const uint32_t at = (p << a.digit_bits) + threadIdx.x;
            total += ALONE ? all[at] & 0xffffu : all[at];
            before += ALONE ? all[at] >> 16 : earlier_blocks[at];
        }
        place = before + wave_exclusive(total, wave_totals);
    }
    __syncthreads();
    if (owner) place += totals_before(wave, wave_totals);
    for (uint32_t tile = 0; tile < a.tiles_per_block; tile++) {
        const uint64_t first = begin + tile * static_cast<uint64_t>(sort_tile);
        if (first >= a.n) break;
        uint2 pair[sort_steps];
        uint32_t rank[sort_steps];
        const uint64_t wave_first = first + wave * 64u * sort_steps + lane;
#pragma unroll
        for (uint32_t s = 0; s < sort_steps; s++) {
            const uint64_t i = wave_first + s * 64u;
            pair[s] = pair_at<I>(a, static_cast<uint32_t>(min(i, static_cast<uint64_t>(a.n - 1))));
        }
        for (uint32_t k = lane; k < digits; k += 64) counts[wave][k] = 0;
        volatile uint16_t* const mine = counts[wave];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (uint32_t s = 0; s < sort_steps; s++) {
            const uint32_t d = digit_of(a, pair[s].x);
            const bool valid = wave_first + s * 64u < a.n;
            uint64_t same = __ballot(valid);  // lanes with the same digit: those that agree with it in every bit
            for (uint32_t b = 0; b < a.digit_bits; b++) {
                const int64_t bit = static_cast<int32_t>(d << (31u - b)) >> 31;  // 0 or all ones
                same &= ~(__ballot(bit != 0) ^ static_cast<uint64_t>(bit));
            }
            const uint32_t earlier = static_cast<uint32_t>(__popcll(same & ((1ull << lane) - 1ull)));
            const uint32_t so_far = mine[d];
            rank[s] = so_far + earlier;
            __builtin_amdgcn_wave_barrier();
            if (valid && earlier == 0) mine[d] = static_cast<uint16_t>(so_far + static_cast<uint32_t>(__popcll(same)));
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        uint32_t in_tile = 0, local = 0;
        if (owner) {
#pragma unroll
            for (uint32_t w = 0; w < sort_waves; w++) in_tile += counts[w][threadIdx.x];
            local = wave_exclusive(in_tile, wave_totals);
        }
        __syncthreads();
        if (owner) {
            local += totals_before(wave, wave_totals);
            to_global[threadIdx.x] = place - local;
            place += in_tile;
#pragma unroll
            for (uint32_t w = 0; w < sort_waves; w++) {
                const uint32_t c = counts[w][threadIdx.x];
                counts[w][threadIdx.x] = static_cast<uint16_t>(local);
                local += c;
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t s = 0; s < sort_steps; s++)
            if (wave_first + s * 64u < a.n) ordered[counts[wave][digit_of(a, pair[s].x)] + rank[s]] = pair[s];
        __syncthreads();
        const uint32_t here = static_cast<uint32_t>(min(static_cast<uint64_t>(sort_tile), a.n - first));
#pragma unroll
        for (uint32_t s = 0; s < sort_steps; s++) {
            const uint32_t k = s * sort_block + threadIdx.x;
            if (k < here) {
                const uint2 p = ordered[k];
                a.out[to_global[digit_of(a, p.x)] + k] = p;
            }
        }
        __syncthreads();
    }
}

// A key's place is the number of smaller keys, and of equal ones before it: 16 keys to a block, each compared by 64 threads
// with a 64th of the list.
template <typename I>
__global__ __launch_bounds__(sort_block) void sort_rank_kernel(SortPass a) {
    __shared__ __attribute__((aligned(16))) uint32_t keys[rank_most];
    __shared__ uint32_t places[sort_block / rank_keys][rank_keys];
    constexpr uint32_t parts = sort_block / rank_keys;
    const uint32_t k = threadIdx.x % rank_keys, part = threadIdx.x / rank_keys;
    const uint32_t per = (a.n + parts * 4 - 1) / (parts * 4) * 4;  // of a part, in fours
    for (uint32_t i = threadIdx.x; i < per * parts; i += sort_block) keys[i] = i < a.n ? key_at<I>(a, i) : 0xffffffffu;
    __syncthreads();
    const uint32_t first = blockIdx.x * rank_keys, i = first + k, mine = keys[min(i, a.n - 1)];
    const uint32_t begin = part * per;
    uint32_t smaller = 0;
    const uint4* const list = reinterpret_cast<const uint4*>(keys + begin);
    if (begin + per <= first || begin >= first + rank_keys) {
        // (equal keys count in the part of the list before the block's keys: as if they were smaller)
        const uint32_t limit = mine + (begin < first ? 1u : 0u);
        for (uint32_t j = 0; j < per / 4; j++) {
            const uint4 other = list[j];
            smaller += (other.x < limit) + (other.y < limit) + (other.z < limit) + (other.w < limit);
        }
    } else {
        for (uint32_t j = 0; j < per; j++) {
            const uint32_t other = keys[begin + j];
            smaller += other < mine + (begin + j < i ? 1u : 0u);
        }
    }
    places[part][k] = smaller;
    __syncthreads();
    if (threadIdx.x < rank_keys && i < a.n) {
        uint32_t to = 0;
        for (uint32_t p = 0; p < parts; p++) to += places[p][k];
        a.out[to] = make_uint2(mine, i);
    }
}

// ---- sums ----------------------------------------------------------------------------------------------------------------

constexpr uint32_t sum_block = 256;
// Items of a group of G lanes: 16 for a wave's (16k indices into 50k rows of 1,024 bfloat16 63 -> 59 us, 60k into 500 rows of 1,000 51 -> 48
// against 8), 8 for fewer lanes, whose block has more of them (8k indices into 30k rows of 256 24.0 us, 24.8 with 16; 1M into 4,096 of 8 floats
// 56.5 and 57.1).
constexpr uint32_t sum_items_of(uint32_t lanes) { return lanes == 64 ? 16 : 8; }

struct SumArgs {
    const uint2* pairs;        // row and position, sorted
    const void* grad_out;
    void* gradient;
    float* heads;              // per block: its first row's piece up to that row's end
    float* tails;              // per block: the sum of the row that is open at its end
    uint32_t* closed;          // per block: 1 where a row ends in it
    uint32_t* first_row;       // per block: the row that is open at its start
    float* chunk_tails;        // long lists, per 64 blocks: the sum of the row that is open at their end
    uint32_t* chunk_closed;    // and 1 where a row ends in them; null: short lists
    uint32_t n, rows, columns;
    uint32_t row_lanes;        // lanes of a row
    uint32_t blocks;
    float scale;
};

// entries among the first `position` items of the merged list, over the wave: 128 places tried a round
__device__ __forceinline__ uint32_t entries_before(const SumArgs& a, uint32_t position) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t lo = position > a.rows ? position - a.rows : 0u, hi = min(position, a.n);
    while (lo < hi) {
        const uint32_t step = (hi - lo + 127u) / 128u, at = lo + lane * step, at2 = at + 64u * step;
        const uint32_t key = a.pairs[min(at, hi - 1)].x, key2 = a.pairs[min(at2, hi - 1)].x;
        const uint32_t before = static_cast<uint32_t>(__popcll(__ballot(at < hi && at + key < position)) + __popcll(__ballot(at2 < hi && at2 + key2 < position)));
        if (before == 0) break;
        hi = min(hi, lo + before * step);
        lo = lo + (before - 1) * step + 1;
    }
    return lo;
}

// G lanes to a row (of a tile of columns). 16k indices into 50k rows of 1,024 bfloat16 read 34 MB and write 102, in 26 us: 5.2 TB/s,
// a large copy's rate.
template <typename T, int W, bool STREAM, int G>
__global__ __launch_bounds__(sum_block) void embedding_sum_kernel(SumArgs a) {
    constexpr uint32_t sum_items = sum_items_of(G), groups = sum_block / G, items = groups * sum_items;
    __shared__ uint32_t s_keys[items], s_values[items], s_start[groups + 1], s_bounds[2];
    __shared__ float s_tail[sum_block / 64][G * W];
    __shared__ uint32_t s_closed[sum_block / 64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t total = a.n + a.rows, first = blockIdx.x * items, last = min(first + items, total);
    if (wave < 2) {
        const uint32_t e = entries_before(a, wave == 0 ? first : last);
        if (lane == 0) s_bounds[wave] = e;
    }
    __syncthreads();
    const uint32_t e0 = s_bounds[0], entries = s_bounds[1] - e0;
    for (uint32_t k = threadIdx.x; k < entries; k += sum_block) {
        const uint2 p = a.pairs[e0 + k];
        s_keys[k] = p.x;
        s_values[k] = p.y;
    }
    __syncthreads();
    for (uint32_t g = threadIdx.x; g <= groups; g += sum_block) {
        const uint32_t position = min(first + g * sum_items, last);
        uint32_t lo = 0, hi = entries;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (e0 + mid + s_keys[mid] < position) lo = mid + 1;
            else hi = mid;
        }
        s_start[g] = lo;
    }
    __syncthreads();

    const uint32_t group = threadIdx.x / G, slot = blockIdx.y * G + threadIdx.x % G, column = min(slot * W, a.columns - W);
    const bool valid = slot < a.row_lanes;
    const uint32_t start = s_start[group], end = s_start[group + 1];
    const uint32_t position = min(first + group * sum_items, last), position_end = min(position + sum_items, last);
    const uint32_t row_start = position - (e0 + start), row_end = position_end - (e0 + end);

    // the group's entries (past its last one, and for indices that count nowhere, some row that is there)
    typename Part<T, W>::type data[sum_items];
    if (entries > 0) {
#pragma unroll
        for (uint32_t k = 0; k < sum_items; k++) {
            const uint32_t e = min(start + k, entries - 1);
            data[k] = load_part<T, W>(static_cast<const T*>(a.grad_out) + static_cast<uint64_t>(s_values[s_keys[e] < a.rows ? e : 0u]) * a.columns + column);
        }
    }

    T* const gradient = static_cast<T*>(a.gradient);
    float sum[W] = {}, head[W] = {};
    bool any_closed = false;
    uint32_t row = row_start;
    auto close = [&]() {
        if (!any_closed) {
#pragma unroll
            for (int j = 0; j < W; j++) head[j] = sum[j];
            any_closed = true;
        } else if (valid) {
            store_part<T, W, STREAM>(gradient + static_cast<uint64_t>(row) * a.columns + column, sum, a.scale);
        }
#pragma unroll
        for (int j = 0; j < W; j++) sum[j] = 0.0f;
        row++;
    };
#pragma unroll
    for (uint32_t k = 0; k < sum_items; k++) {
        if (start + k < end) {
            const uint32_t key = s_keys[start + k];
            while (row < key && row < row_end) close();
            // (entries of indices that count nowhere stand behind the last row's end: their sums go nowhere)
#pragma unroll
            for (int j = 0; j < W; j++) sum[j] += value_of<T, W>(data[k], j);
        }
    }
    while (row < row_end) close();

    // what is open at the start of each group: a segmented scan of the groups' open sums, first over the wave, then over the block
    float scanned[W];
    uint32_t flag = any_closed ? 1u : 0u;
#pragma unroll
    for (int j = 0; j < W; j++) scanned[j] = sum[j];
#pragma unroll
    for (uint32_t o = G; o < 64; o <<= 1) {
        const uint32_t other_flag = __shfl_up(flag, o);
#pragma unroll
        for (int j = 0; j < W; j++) {
            const float other = __shfl_up(scanned[j], o);
            if (lane >= o && !flag) scanned[j] += other;
        }
        if (lane >= o) flag |= other_flag;
    }
    if (lane >= 64 - G) {
#pragma unroll
        for (int j = 0; j < W; j++) s_tail[wave][(lane % G) * W + j] = scanned[j];
        if (lane == 63) s_closed[wave] = flag;
    }
    __syncthreads();
    uint32_t before_flag = 0, block_flag = 0;
    float before[W] = {}, block_tail[W] = {};
#pragma unroll
    for (uint32_t w = 0; w < sum_block / 64; w++) {
        if (w == wave) {
            before_flag = block_flag;
#pragma unroll
            for (int j = 0; j < W; j++) before[j] = block_tail[j];
        }
        const bool closed = s_closed[w] != 0;
#pragma unroll
        for (int j = 0; j < W; j++) block_tail[j] = s_tail[w][(lane % G) * W + j] + (closed ? 0.0f : block_tail[j]);
        block_flag |= closed ? 1u : 0u;
    }
    if constexpr (G < 64) {
        const uint32_t wave_flag = __shfl_up(flag, G);
#pragma unroll
        for (int j = 0; j < W; j++) {
            const float other = __shfl_up(scanned[j], G);
            if (lane >= G) before[j] = other + (wave_flag ? 0.0f : before[j]);
        }
        if (lane >= G) before_flag |= wave_flag;
    }
    const uint64_t piece = (static_cast<uint64_t>(blockIdx.x) * gridDim.y * G + slot) * W;
    if (any_closed) {
#pragma unroll
        for (int j = 0; j < W; j++) head[j] += before[j];
        if (!before_flag) {
#pragma unroll
            for (int j = 0; j < W; j++) a.heads[piece + j] = head[j];
        } else if (valid) {
            store_part<T, W, STREAM>(gradient + static_cast<uint64_t>(row_start) * a.columns + column, head, a.scale);
        }
    }
    if (threadIdx.x < G) {
#pragma unroll
        for (int j = 0; j < W; j++) a.tails[piece + j] = block_tail[j];
    }
    if (threadIdx.x == 0 && blockIdx.y == 0) {
        a.closed[blockIdx.x] = block_flag;
        a.first_row[blockIdx.x] = first - e0;
    }
}

constexpr uint32_t join_block = 256, chunk = 64;
// Blocks of the sums from which the chunks have a kernel of their own, which costs 2.5 to 9 us: without and with it, us, 130k indices into 40 rows of
// 2,048 bfloat16 (2,032 blocks) 157 and 166 over even rows, 198 and 165 where one row has half of them, 225 and 155 where it has all; 200k into 50k
// of 1,024 (3,907) 136 and 139, 181 and 150, 212 and 143; 200k into 50k of 256 floats 75 and 77, 102 and 83, 125 and 82; 200k into 3,000 of 1,024
// bfloat16 113 and 116, 161 and 122, 189 and 116. Even rows pay 2 to 6 % for it; just below the limit a row that has all pays 45 % without it.
constexpr uint32_t chunks_from = 2048;

// The last of closed[floor, at) that is set, or floor and `found` unset. Every wave looks at 256 at once.
__device__ __forceinline__ uint32_t last_closed(const uint32_t* closed, uint32_t floor, uint32_t at, bool& found) {
    const uint32_t lane = threadIdx.x & 63u;
    while (at > floor) {
        uint32_t flag[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) flag[j] = closed[max(at, floor + 1u + j * 64u + lane) - 1u - j * 64u - lane];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint64_t ends = __ballot(j * 64u + lane < at - floor && flag[j] != 0);
            if (ends) {
                found = true;
                return at - j * 64u - static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(ends)));
            }
        }
        at = at - floor > 256 ? at - 256 : floor;
    }
    return floor;
}

// adds what this thread's part of the block has of tails[from, to)
template <int W, int G>
__device__ __forceinline__ void add_tails(const float* tails, uint64_t stride, uint32_t from, uint32_t to, float* sum) {
#pragma unroll 8
    for (uint32_t k = from + threadIdx.x / G; k < to; k += join_block / G) {
#pragma unroll
        for (int j = 0; j < W; j++) sum[j] += tails[k * stride + j];
    }
}

// the sum over the block's parts, in its first G threads
template <int W, int G>
__device__ __forceinline__ void sum_parts(float* sum) {
    __shared__ float parts[join_block / 64][G * W];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
    for (uint32_t o = G; o < 64; o <<= 1) {
#pragma unroll
        for (int j = 0; j < W; j++) sum[j] += __shfl_xor(sum[j], o);
    }
    if (lane < G) {
#pragma unroll
        for (int j = 0; j < W; j++) parts[wave][lane * W + j] = sum[j];
    }
    __syncthreads();
    if (threadIdx.x >= G) return;
#pragma unroll
    for (uint32_t w = 1; w < join_block / 64; w++)
#pragma unroll
        for (int j = 0; j < W; j++) sum[j] += parts[w][lane * W + j];
}

// Long lists: what is open at the end of every 64 blocks.
template <int W, int G>
__global__ __launch_bounds__(join_block) void embedding_chunk_kernel(SumArgs a) {
    const uint32_t lane = threadIdx.x & 63u, first = blockIdx.x * chunk, count = min(chunk, a.blocks - first);
    const uint64_t ends = __ballot(lane < count && a.closed[first + min(lane, count - 1u)] != 0);
    const uint32_t from = ends ? first + 63u - static_cast<uint32_t>(__clzll(ends)) : first;
    const uint32_t slot = blockIdx.y * G + threadIdx.x % G;
    const uint64_t stride = static_cast<uint64_t>(gridDim.y) * G * W, piece = static_cast<uint64_t>(slot) * W;
    float sum[W] = {};
    add_tails<W, G>(a.tails + piece, stride, from, first + count, sum);
    sum_parts<W, G>(sum);
    if (threadIdx.x < G) {
#pragma unroll
        for (int j = 0; j < W; j++) a.chunk_tails[blockIdx.x * stride + piece + j] = sum[j];
    }
    if (threadIdx.x == 0 && blockIdx.y == 0) a.chunk_closed[blockIdx.x] = ends != 0;
}

// A block per block of the sums and tile of columns: the row that was open at that block's start, if it ends there, from
// the open sums of the blocks before it since the last end of a row, and the block's own first piece. In long lists the blocks
// of earlier chunks stand summed, so that a row that most indices name is two short chains. (One wave, one block
// of the sums after another, took 397 us for 200k indices of one row of 1,024 bfloat16 where even rows took 135; 143 now, 139 even.)
template <typename T, int W, bool STREAM, int G>
__global__ __launch_bounds__(join_block) void embedding_join_kernel(SumArgs a) {
    const uint32_t b = blockIdx.x;
    if (!a.closed[b]) return;
    const uint32_t slot = blockIdx.y * G + threadIdx.x % G;
    const uint64_t stride = static_cast<uint64_t>(gridDim.y) * G * W, piece = static_cast<uint64_t>(slot) * W;
    float sum[W] = {};
    bool found = false;
    const uint32_t from = last_closed(a.closed, a.chunk_closed ? b / chunk * chunk : 0u, b, found);
    add_tails<W, G>(a.tails + piece, stride, from, b, sum);
    if (a.chunk_closed && !found) add_tails<W, G>(a.chunk_tails + piece, stride, last_closed(a.chunk_closed, 0u, b / chunk, found), b / chunk, sum);
    sum_parts<W, G>(sum);
    if (threadIdx.x < G && slot < a.row_lanes) {
#pragma unroll
        for (int j = 0; j < W; j++) sum[j] += a.heads[b * stride + piece + j];
        store_part<T, W, STREAM>(static_cast<T*>(a.gradient) + static_cast<uint64_t>(a.first_row[b]) * a.columns + min(slot * W, a.columns - W), sum, a.scale);
    }
}

// W floats (one or fours) of a partial table
template <int W>
__device__ __forceinline__ void store_floats(float* p, const float* x) {
    if constexpr (W == 1) {
        *p = x[0];
    } else {
#pragma unroll
        for (int j = 0; j < W; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
    }
}

template <int W>
__device__ __forceinline__ void load_floats(const float* p, float* x) {
    if constexpr (W == 1) {
        x[0] = *p;
    } else {
#pragma unroll
        for (int j = 0; j < W; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + j);
            x[j] = v.x;
            x[j + 1] = v.y;
            x[j + 2] = v.z;
            x[j + 3] = v.w;
        }
    }
}

// ---- small tables ----------------------------------------------------------------------------------------------------------
// A small table needs no list in order over the GPU: a block sorts a tile of the indices in LDS, sums its runs and writes a partial
// table of its own (every row, in 32 bits), and a second kernel adds the partial tables up. grad_out is read a tile at a time,
// where the long list's runs gather rows from all over it, 128-byte lines for 32 bytes; two launches stand for five to seven. What it
// costs is the partial tables, written and read once, so they decide: at most 32 MB of them, 256 KB each (us by the list and by tiles: 1M
// indices into 4,096 rows of 8 floats, 32 MB, 57 and 37, of 8 bfloat16 56 and 43; 200k into 257 rows of 45 30 and 20, 20k into 500 of 8 18 and 11; past that 100k
// into 4,096 rows of 64 28 and 46, 200k into 700 rows of 64, 35 MB, 31 and 33, 4,000 into 4,096 rows of 64, 1 MB each, 14 and 23).
// The bytes are where rows of 64 floats cross. Narrow rows cross later, past 8,192 rows, and pay the list's price from 4,097 on: 1M
// into 5,000 rows of 8 floats 58 and 39, 8,192 57 and 45, 16,384 63 and 65, 32,768 64 and 124; 16,384 rows of 4 62 and 46; 100k
// into 5,000 rows of 8 27 and 19, 16,384 31 and 31, 8,192 rows of 16 27 and 31; 1M into 8,192 of 8 bfloat16 56 and 52.

constexpr uint32_t tile_rows = 4096, tile_lanes = 16, tile_position_bits = 12;
constexpr uint32_t tile_most_blocks = 256;
constexpr uint64_t tile_most_bytes = 32ull << 20, tile_table_bytes = 256ull << 10;
constexpr uint32_t tables_block = 256, tables_parts = 8, tables_lanes = tables_block / tables_parts;

struct TileSumArgs {
    SortPass keys;             // indices, n, rows, padding, tiles_per_block; digit_bits of a local pass
    uint32_t passes;
    const void* grad_out;
    float* partials;           // blocks x rows x lanes x lane's values
    uint32_t columns, row_lanes, index_bytes;
};

// Groups of G lanes take the ordered entries evenly, whatever the runs; the group that holds a run's last entry writes its sum, with what
// earlier groups had of it by a segmented scan. Rows that no entry meets keep the zeros that the block wrote first. A block's chain of
// steps bounds it, one block of 1,024 threads to a CU with nothing beside it: 1M indices into 4,096 rows of 8 floats take 31 us (35 over even
// rows), and of a block's cycles 39 % went to the tile's sort, 31 % to loads and sums, 17 % to the scan (read at one block). The tables' sum takes 7.
template <typename T, int W, int G, uint32_t STEPS>
__global__ __launch_bounds__(sort_block) void embedding_tile_sum_kernel(TileSumArgs a) {
    constexpr uint32_t tile_size = sort_block * STEPS, groups = sort_block / G, batch = 8;
    struct Sorting {
        uint16_t counts[sort_waves][sort_most_digits];
        uint32_t wave_totals[sort_waves];
    };
    struct Summing {
        uint32_t closed[sort_waves];
        float tail[sort_waves][G * W];
    };
    __shared__ uint32_t ordered[tile_size];  // row << 12 | position in the tile, in order of rows
    __shared__ __attribute__((aligned(16))) unsigned char shared[sizeof(Sorting) > sizeof(Summing) ? sizeof(Sorting) : sizeof(Summing)];
    Sorting& sorting = *reinterpret_cast<Sorting*>(shared);
    Summing& summing = *reinterpret_cast<Summing*>(shared);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, rows = a.keys.rows;
    const uint32_t digits = 1u << a.keys.digit_bits;
    const uint32_t group = threadIdx.x / G, slot = threadIdx.x % G, column = min(slot * W, a.columns - W);
    const bool valid = slot < a.row_lanes;
    float* const table = a.partials + static_cast<uint64_t>(blockIdx.x) * rows * a.row_lanes * W;
    const float zeros[W] = {};
    for (uint32_t k = threadIdx.x; k < rows * a.row_lanes; k += sort_block) store_floats<W>(table + static_cast<uint64_t>(k) * W, zeros);

    for (uint32_t tile = 0; tile < a.keys.tiles_per_block; tile++) {
        const uint64_t first = (static_cast<uint64_t>(blockIdx.x) * a.keys.tiles_per_block + tile) * tile_size;
        const uint32_t here = first >= a.keys.n ? 0u : static_cast<uint32_t>(min(static_cast<uint64_t>(tile_size), a.keys.n - first));
        if (tile > 0 && here == 0) break;
        const uint32_t mine = wave * 64u * STEPS + lane;
        uint32_t x[STEPS], rank[STEPS];
        auto load_keys = [&](auto index) {
            using I = decltype(index);
#pragma unroll
            for (uint32_t s = 0; s < STEPS; s++) {
                const uint32_t k = mine + s * 64u;
                x[s] = key_at<I>(a.keys, static_cast<uint32_t>(min(first + k, static_cast<uint64_t>(a.keys.n - 1)))) << tile_position_bits | k;
            }
        };
        if (a.index_bytes == 4) load_keys(int32_t{});
        else load_keys(int64_t{});
        for (uint32_t pass = 0; pass < a.passes; pass++) {
            const uint32_t shift = tile_position_bits + pass * a.keys.digit_bits;
            if (pass > 0) {
#pragma unroll
                for (uint32_t s = 0; s < STEPS; s++) x[s] = ordered[mine + s * 64u];
            }
            for (uint32_t k = lane; k < digits; k += 64) sorting.counts[wave][k] = 0;
            volatile uint16_t* const counts = sorting.counts[wave];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (uint32_t s = 0; s < STEPS; s++) {
                const uint32_t d = (x[s] >> shift) & (digits - 1u);
                const bool in = mine + s * 64u < here;
                uint64_t same = __ballot(in);
                for (uint32_t b = 0; b < a.keys.digit_bits; b++) {
                    const int64_t bit = static_cast<int32_t>(d << (31u - b)) >> 31;
                    same &= ~(__ballot(bit != 0) ^ static_cast<uint64_t>(bit));
                }
                const uint32_t earlier = static_cast<uint32_t>(__popcll(same & ((1ull << lane) - 1ull)));
                const uint32_t so_far = counts[d];
                rank[s] = so_far + earlier;
                __builtin_amdgcn_wave_barrier();
                if (in && earlier == 0) counts[d] = static_cast<uint16_t>(so_far + static_cast<uint32_t>(__popcll(same)));
                __builtin_amdgcn_wave_barrier();
            }
            __syncthreads();
            const bool owner = threadIdx.x < digits;
            uint32_t local = 0;
            if (owner) {
                uint32_t in_tile = 0;
#pragma unroll
                for (uint32_t w = 0; w < sort_waves; w++) in_tile += sorting.counts[w][threadIdx.x];
                local = wave_exclusive(in_tile, sorting.wave_totals);
            }
            __syncthreads();
            if (owner) {
                local += totals_before(wave, sorting.wave_totals);
#pragma unroll
                for (uint32_t w = 0; w < sort_waves; w++) {
                    const uint32_t c = sorting.counts[w][threadIdx.x];
                    sorting.counts[w][threadIdx.x] = static_cast<uint16_t>(local);
                    local += c;
                }
            }
            __syncthreads();
#pragma unroll
            for (uint32_t s = 0; s < STEPS; s++)
                if (mine + s * 64u < here) ordered[sorting.counts[wave][(x[s] >> shift) & (digits - 1u)] + rank[s]] = x[s];
            __syncthreads();
        }

        // the entries that count, evenly over the groups
        uint32_t entries = here;
        for (uint32_t lo = 0; lo < entries;) {
            const uint32_t mid = (lo + entries) / 2;
            if (ordered[mid] >> tile_position_bits < rows) lo = mid + 1;
            else entries = mid;
        }
        const uint32_t per_group = (entries + groups - 1) / groups;
        const uint32_t start = min(group * per_group, entries), end = min(start + per_group, entries);
        float sum[W] = {}, head[W] = {};
        bool any_closed = false;
        uint32_t head_row = 0;
        auto write = [&](uint32_t row, const float* values) {
            if (!valid) return;
            float* const at = table + (static_cast<uint64_t>(row) * a.row_lanes + slot) * W;
            if (tile == 0) {
                store_floats<W>(at, values);
            } else {
                float old[W];
                load_floats<W>(at, old);
#pragma unroll
                for (int j = 0; j < W; j++) old[j] += values[j];
                store_floats<W>(at, old);
            }
        };
        for (uint32_t from = start; from < end; from += batch) {
            typename Part<T, W>::type data[batch];
            uint32_t key[batch + 1];
#pragma unroll
            for (uint32_t k = 0; k <= batch; k++) {
                const uint32_t entry = ordered[min(from + k, entries - 1)];
                key[k] = from + k < entries ? entry >> tile_position_bits : rows;
                if (k == batch) break;
                const uint64_t i = first + (entry & ((1u << tile_position_bits) - 1u));
                data[k] = load_part<T, W>(static_cast<const T*>(a.grad_out) + i * a.columns + column);
            }
#pragma unroll
            for (uint32_t k = 0; k < batch; k++) {
                if (from + k < end) {
#pragma unroll
                    for (int j = 0; j < W; j++) sum[j] += value_of<T, W>(data[k], j);
                    if (key[k] != key[k + 1]) {  // the run's last entry
                        if (any_closed) {
                            write(key[k], sum);
                        } else {
                            any_closed = true;
                            head_row = key[k];
#pragma unroll
                            for (int j = 0; j < W; j++) head[j] = sum[j];
                        }
#pragma unroll
                        for (int j = 0; j < W; j++) sum[j] = 0.0f;
                    }
                }
            }
        }

        // the run that is open at each group's start: the segmented scan of the groups' open sums
        float scanned[W];
        uint32_t flag = any_closed ? 1u : 0u;
#pragma unroll
        for (int j = 0; j < W; j++) scanned[j] = sum[j];
#pragma unroll
        for (uint32_t o = G; o < 64; o <<= 1) {
            const uint32_t other_flag = __shfl_up(flag, o);
#pragma unroll
            for (int j = 0; j < W; j++) {
                const float other = __shfl_up(scanned[j], o);
                if (lane >= o && !flag) scanned[j] += other;
            }
            if (lane >= o) flag |= other_flag;
        }
        if (lane >= 64 - G) {
#pragma unroll
            for (int j = 0; j < W; j++) summing.tail[wave][(lane % G) * W + j] = scanned[j];
            if (lane == 63) summing.closed[wave] = flag;
        }
        __syncthreads();
        float before[W] = {};
        for (uint32_t w = 0; w < wave; w++) {
            const bool closed = summing.closed[w] != 0;
#pragma unroll
            for (int j = 0; j < W; j++) before[j] = summing.tail[w][(lane % G) * W + j] + (closed ? 0.0f : before[j]);
        }
        if constexpr (G < 64) {
            const uint32_t wave_flag = __shfl_up(flag, G);
#pragma unroll
            for (int j = 0; j < W; j++) {
                const float other = __shfl_up(scanned[j], G);
                if (lane >= G) before[j] = other + (wave_flag ? 0.0f : before[j]);
            }
        }
        if (any_closed) {
#pragma unroll
            for (int j = 0; j < W; j++) head[j] += before[j];
            write(head_row, head);
        }
        __syncthreads();  // (before the next tile's sort writes where the sums were read)
    }
}

// The partial tables' sum, eight threads to a lane of a row, each every eighth table: a fixed order.
template <typename T, int W>
__global__ __launch_bounds__(tables_block) void embedding_tables_kernel(const float* __restrict__ partials, T* __restrict__ gradient, uint32_t tables, uint32_t rows,
                                                               uint32_t row_lanes, uint32_t columns, float scale) {
    __shared__ float s_sum[tables_parts][tables_lanes][W];
    const uint32_t part = threadIdx.x / tables_lanes, k = threadIdx.x % tables_lanes, count = rows * row_lanes;
    const uint32_t at = blockIdx.x * tables_lanes + k, safe = min(at, count - 1);
    const float* const from = partials + static_cast<uint64_t>(safe) * W;
    const uint64_t stride = static_cast<uint64_t>(count) * W;
    float sum[W] = {};
#pragma unroll 8
    for (uint32_t t = part; t < tables; t += tables_parts) {
        float x[W];
        load_floats<W>(from + t * stride, x);
#pragma unroll
        for (int j = 0; j < W; j++) sum[j] += x[j];
    }
#pragma unroll
    for (int j = 0; j < W; j++) s_sum[part][k][j] = sum[j];
    __syncthreads();
    if (part != 0 || at >= count) return;
#pragma unroll
    for (uint32_t p = 1; p < tables_parts; p++)
#pragma unroll
        for (int j = 0; j < W; j++) sum[j] += s_sum[p][k][j];
    const uint32_t row = at / row_lanes, slot = at - row * row_lanes;
    store_part<T, W, false>(gradient + static_cast<uint64_t>(row) * columns + min(slot * W, columns - W), sum, scale);
}

uint32_t bit_width(uint32_t x) { return x == 0 ? 0u : 32u - static_cast<uint32_t>(__builtin_clz(x)); }

int lane_values(const EmbeddingArgs& a) {
    const uint32_t full = a.type == type_float ? 4 : 8;
    return a.columns >= full ? static_cast<int>(full) : 1;
}

uint32_t lanes_of_row(const EmbeddingArgs& a) { return div_up(a.columns, static_cast<uint32_t>(lane_values(a))); }

uint64_t output_bytes(const EmbeddingArgs& a, uint64_t rows) { return rows * a.columns * (a.type == type_float ? 4 : 2); }

// f(a value of the type, the lane's values, whether an output of so many rows is stored past the caches), the latter two as constants
template <typename F>
void with_type(const EmbeddingArgs& a, uint64_t output_rows, F&& f) {
    const bool one = lane_values(a) == 1, stream = output_bytes(a, output_rows) >= stream_from;
    auto widths = [&](auto t) {
        constexpr int full = 16 / sizeof(t);
        if (one) f(t, std::integral_constant<int, 1>{}, std::false_type{});
        else if (stream) f(t, std::integral_constant<int, full>{}, std::true_type{});
        else f(t, std::integral_constant<int, full>{}, std::false_type{});
    };
    if (a.type == type_float) widths(float{});
    else if (a.type == type_bfloat16) widths(__bf16{});
    else widths(_Float16{});
}

// lanes of a group: the power of two that holds a row, or a wave
uint32_t group_lanes(const EmbeddingArgs& a) {
    uint32_t g = 1;
    while (g < 64 && g < lanes_of_row(a)) g *= 2;
    return g;
}

uint32_t sum_blocks(const EmbeddingArgs& a) { return div_up(static_cast<uint64_t>(a.n) + a.rows, sum_block / group_lanes(a) * sum_items_of(group_lanes(a))); }

uint32_t sort_blocks(const SortPass& p) { return div_up(p.n, static_cast<uint64_t>(sort_block) * p.steps * p.tiles_per_block); }

// Digits, tiles and steps of a list's passes. A block reads the whole table, blocks x digits, so both are held against it: as few
// passes as digits of 9 bits make, 8 bits past 128 blocks of four keys a thread; and one key a thread, in four times the blocks, where the
// table has at most 32,768 entries then (us with four and one: 33k indices into 5,000 rows 31 and 26, 130k 33 and 28, 200k 35 and 32.5; past
// that 100k into 100,000 rows 36 and 38, 200k into 257 25 and 28).
void plan_sort(SortPass& p) {
    p.steps = sort_steps_most;
    p.tiles_per_block = div_up(div_up(p.n, sort_block * p.steps), sort_max_blocks);
    const uint32_t bits = bit_width(p.rows), most = sort_blocks(p) > 128 ? sort_most_bits - 1 : sort_most_bits;
    p.digit_bits = std::max(div_up(bits, div_up(bits, most)), sort_least_bits);
    if (div_up(p.n, sort_block) << p.digit_bits <= 32768) p.steps = p.tiles_per_block = 1;
}

template <typename I>
void launch_sort_pass(const SortPass& p, hipStream_t s) {
    const uint32_t blocks = sort_blocks(p);
    if (p.n <= sort_alone && p.steps == 1) {
        sort_scatter_kernel<I, true, 1><<<blocks, sort_block, 0, s>>>(p);
    } else if (p.steps == 1) {
        sort_count_kernel<I, 1><<<blocks, sort_block, 0, s>>>(p);
        sort_scatter_kernel<I, false, 1><<<blocks, sort_block, 0, s>>>(p);
    } else {
        sort_count_kernel<I, 4><<<blocks, sort_block, 0, s>>>(p);
        sort_scatter_kernel<I, false, 4><<<blocks, sort_block, 0, s>>>(p);
    }
}

// The blocks and tiles of a small table's gradient; no blocks where the table is not small.
struct TilePlan {
    uint32_t blocks = 0, steps = 1, tiles_per_block = 1;
    uint64_t bytes = 0;  // of the partial tables
};

TilePlan plan_tiles(const EmbeddingArgs& a) {
    TilePlan p;
    if (a.n == 0 || a.rows > tile_rows || lanes_of_row(a) > tile_lanes) return p;
    // (one key a thread up to 262,144 indices, so that there are blocks for the GPU; then two, four, and more tiles to a block)
    const uint32_t pieces = div_up(a.n, sort_block);
    p.steps = pieces <= tile_most_blocks ? 1 : pieces <= 2 * tile_most_blocks ? 2 : 4;
    const uint32_t tiles = div_up(pieces, p.steps);
    p.tiles_per_block = div_up(tiles, tile_most_blocks);
    p.blocks = div_up(tiles, p.tiles_per_block);
    const uint64_t table = static_cast<uint64_t>(a.rows) * lanes_of_row(a) * static_cast<uint64_t>(lane_values(a)) * 4;
    p.bytes = p.blocks * table;
    if (table > tile_table_bytes || p.bytes > tile_most_bytes) p.blocks = 0;
    return p;
}

template <typename T, int W, int G>
void launch_tiles(const TileSumArgs& a, const TilePlan& p, hipStream_t s) {
    if (p.steps == 1) embedding_tile_sum_kernel<T, W, G, 1><<<p.blocks, sort_block, 0, s>>>(a);
    else if (p.steps == 2) embedding_tile_sum_kernel<T, W, G, 2><<<p.blocks, sort_block, 0, s>>>(a);
    else embedding_tile_sum_kernel<T, W, G, 4><<<p.blocks, sort_block, 0, s>>>(a);
}

bool launch_small_table(const EmbeddingArgs& a, const TilePlan& p, const void* grad_out, uint32_t padding, void* gradient, float* partials, hipStream_t s) {
    TileSumArgs t{};  // (of t.keys the tile kernel reads what is set here)
    t.keys.indices = a.indices;
    t.keys.n = a.n;
    t.keys.rows = a.rows;
    t.keys.padding = padding;
    t.keys.tiles_per_block = p.tiles_per_block;
    const uint32_t bits = bit_width(a.rows);
    t.passes = bits > sort_most_bits ? 2 : 1;
    t.keys.digit_bits = std::max(div_up(bits, t.passes), sort_least_bits);
    t.grad_out = grad_out;
    t.partials = partials;
    t.columns = a.columns;
    t.row_lanes = lanes_of_row(a);
    t.index_bytes = static_cast<uint32_t>(a.index_bytes);
    with_type(a, 0, [&](auto v, auto w, auto) {
        using T = decltype(v);
        constexpr int W = decltype(w)::value;
        switch (group_lanes(a)) {
            case 1: launch_tiles<T, W, 1>(t, p, s); break;
            case 2: launch_tiles<T, W, 2>(t, p, s); break;
            case 4: launch_tiles<T, W, 4>(t, p, s); break;
            case 8: launch_tiles<T, W, 8>(t, p, s); break;
            default:
                if constexpr (W > 1) launch_tiles<T, W, 16>(t, p, s);
        }
        const uint32_t blocks = div_up(static_cast<uint64_t>(a.rows) * t.row_lanes, tables_lanes);
        embedding_tables_kernel<T, W><<<blocks, tables_block, 0, s>>>(partials, static_cast<T*>(gradient), p.blocks, a.rows, t.row_lanes, a.columns, a.scale);
    });
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

struct GradientLayout {
    uint2* pairs[2];
    uint32_t* table;
    float* heads;
    float* tails;
    uint32_t* closed;
    uint32_t* first_row;
    float* chunk_tails = nullptr;
    uint32_t* chunk_closed = nullptr;
    size_t bytes;

    static GradientLayout carve(char* base, const EmbeddingArgs& a) {
        GradientLayout l;
        size_t used = 0;
        auto take = [&](size_t bytes) {
            char* p = base + used;
            used += (bytes + 255) / 256 * 256;
            return p;
        };
        const size_t lanes = group_lanes(a), blocks = sum_blocks(a);
        const size_t piece = div_up(lanes_of_row(a), lanes) * lanes * static_cast<size_t>(lane_values(a)) * 4;
        for (int k = 0; k < 2; k++) l.pairs[k] = reinterpret_cast<uint2*>(take(size_t{a.n} * 8));
        l.table = reinterpret_cast<uint32_t*>(take(size_t{sort_max_blocks} * sort_most_digits * 4));
        l.heads = reinterpret_cast<float*>(take(blocks * piece));
        l.tails = reinterpret_cast<float*>(take(blocks * piece));
        l.closed = reinterpret_cast<uint32_t*>(take(blocks * 4));
        l.first_row = reinterpret_cast<uint32_t*>(take(blocks * 4));
        if (blocks > chunks_from) {
            l.chunk_tails = reinterpret_cast<float*>(take(div_up(blocks, chunk) * piece));
            l.chunk_closed = reinterpret_cast<uint32_t*>(take(size_t{div_up(blocks, chunk)} * 4));
        }
        l.bytes = used;
        return l;
    }
};

template <typename T, int W, bool STREAM, int G>
void launch_sums(const SumArgs& a, hipStream_t s) {
    const uint32_t tiles = div_up(a.row_lanes, G);
    embedding_sum_kernel<T, W, STREAM, G><<<dim3(a.blocks, tiles), sum_block, 0, s>>>(a);
    if (a.chunk_closed) embedding_chunk_kernel<W, G><<<dim3(div_up(a.blocks, chunk), tiles), join_block, 0, s>>>(a);
    embedding_join_kernel<T, W, STREAM, G><<<dim3(a.blocks, tiles), join_block, 0, s>>>(a);
}

}  // namespace

bool launch_embedding_lookup(const EmbeddingArgs& a, const void* table, uint64_t row_stride, void* out, hipStream_t s) {
    if (a.n == 0 || a.columns == 0) return true;
    if (a.rows == 0) {
        const uint64_t values = static_cast<uint64_t>(a.n) * a.columns;
        const uint32_t blocks = values > 2048ull * lookup_block ? 2048u : div_up(values, lookup_block);
        with_type(a, a.n, [&](auto t, auto, auto) {
            using T = decltype(t);
            embedding_zero_kernel<T><<<blocks, lookup_block, 0, s>>>(static_cast<T*>(out), values);
        });
        EFGS_HIP_CHECK(hipGetLastError());
        return true;
    }
    LookupArgs l;
    l.indices = a.indices;
    l.table = table;
    l.out = out;
    l.row_stride = row_stride;
    l.n = a.n;
    l.rows = a.rows;
    l.columns = a.columns;
    l.row_lanes = lanes_of_row(a);
    l.lanes = l.row_lanes < lookup_tile ? l.row_lanes : lookup_tile;
    l.lanes_rcp = (1u << 20) / l.lanes + 1;
    l.rows_per_block = lookup_tile / l.lanes;
    l.scale = a.scale;
    const uint64_t blocks = div_up(a.n, l.rows_per_block);
    for (uint64_t b = 0; b < blocks; b += max_blocks) {
        l.first = static_cast<uint32_t>(b * l.rows_per_block);
        const dim3 grid(static_cast<uint32_t>(blocks - b < max_blocks ? blocks - b : max_blocks), div_up(l.row_lanes, lookup_tile));
        with_type(a, a.n, [&](auto t, auto w, auto stream) {
            using T = decltype(t);
            constexpr int W = decltype(w)::value;
            constexpr bool S = decltype(stream)::value;
            if (a.index_bytes == 4) embedding_lookup_kernel<T, W, S, int32_t><<<grid, lookup_block, 0, s>>>(l);
            else embedding_lookup_kernel<T, W, S, int64_t><<<grid, lookup_block, 0, s>>>(l);
        });
        EFGS_HIP_CHECK(hipGetLastError());
    }
    return true;
}

bool embedding_gradient_fits(const EmbeddingArgs& a) {
    return static_cast<uint64_t>(a.n) + a.rows <= 0xffff0000ull && sum_blocks(a) <= max_blocks;
}

size_t embedding_gradient_bytes(const EmbeddingArgs& a) {
    const TilePlan tiles = plan_tiles(a);
    return tiles.blocks > 0 ? static_cast<size_t>(tiles.bytes) : GradientLayout::carve(nullptr, a).bytes;
}

bool launch_embedding_gradient(const EmbeddingArgs& a, const void* grad_out, uint32_t padding, void* gradient, void* workspace, hipStream_t s) {
    if (a.rows == 0 || a.columns == 0) return true;
    const TilePlan tiles = plan_tiles(a);
    if (tiles.blocks > 0) return launch_small_table(a, tiles, grad_out, padding, gradient, static_cast<float*>(workspace), s);
    const GradientLayout l = GradientLayout::carve(static_cast<char*>(workspace), a);
    uint32_t current = 0;
    if (a.n > 0) {
        SortPass p;
        p.indices = a.indices;
        p.in = nullptr;
        p.out = l.pairs[0];
        p.table = l.table;
        p.n = a.n;
        p.rows = a.rows;
        p.padding = padding;
        p.shift = 0;
        if (a.n <= rank_most) {
            const uint32_t blocks = div_up(a.n, rank_keys);
            if (a.index_bytes == 4) sort_rank_kernel<int32_t><<<blocks, sort_block, 0, s>>>(p);
            else sort_rank_kernel<int64_t><<<blocks, sort_block, 0, s>>>(p);
        } else {
            plan_sort(p);
            const uint32_t passes = div_up(bit_width(a.rows), p.digit_bits);
            if (a.index_bytes == 4) launch_sort_pass<int32_t>(p, s);
            else launch_sort_pass<int64_t>(p, s);
            for (uint32_t k = 1; k < passes; k++) {
                p.shift = k * p.digit_bits;
                p.in = l.pairs[current];
                current ^= 1u;
                p.out = l.pairs[current];
                launch_sort_pass<uint2>(p, s);
            }
        }
        EFGS_HIP_CHECK(hipGetLastError());
    }
    SumArgs u;
    u.pairs = l.pairs[current];
    u.grad_out = grad_out;
    u.gradient = gradient;
    u.heads = l.heads;
    u.tails = l.tails;
    u.closed = l.closed;
    u.first_row = l.first_row;
    u.chunk_tails = l.chunk_tails;
    u.chunk_closed = l.chunk_closed;
    u.n = a.n;
    u.rows = a.rows;
    u.columns = a.columns;
    u.row_lanes = lanes_of_row(a);
    u.blocks = sum_blocks(a);
    u.scale = a.scale;
    with_type(a, a.rows, [&](auto t, auto w, auto stream) {
        using T = decltype(t);
        constexpr int W = decltype(w)::value;
        constexpr bool S = decltype(stream)::value;
        switch (group_lanes(a)) {
            case 1: launch_sums<T, W, S, 1>(u, s); break;
            case 2: launch_sums<T, W, S, 2>(u, s); break;
            case 4: launch_sums<T, W, S, 4>(u, s); break;
            default:
                if constexpr (W == 1) {
                    launch_sums<T, W, S, 8>(u, s);  // (at most 7 lanes of one value)
                } else {
                    switch (group_lanes(a)) {
                        case 8: launch_sums<T, W, S, 8>(u, s); break;
                        case 16: launch_sums<T, W, S, 16>(u, s); break;
                        case 32: launch_sums<T, W, S, 32>(u, s); break;
                        default: launch_sums<T, W, S, 64>(u, s); break;
                    }
                }
        }
    });
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

}  // namespace efgs
