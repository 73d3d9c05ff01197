// The cross entropy's matrix products above 64 columns, on v_mfma_f32_16x16x32: 256 x 256 results to a block of eight waves (2 along i, 4 along j,
// 128 x 64 each), or, where those would leave most of the GPU idle, 128 x 128 to one of four (64 x 64 each); 64 of k at a time.
//
// Floats are multiplied as three bfloat16 parts (their sum is the float to 2^-26 of it), by the six pairs of parts that matter, one pair's steps after
// another's. Six products on this instruction take 6 / 16 of the matrix unit's time that one takes on v_mfma_f32_16x16x4_f32.
//
// Operand tiles go from memory to LDS past the registers (16 bytes a lane), two stages of 64 KB (32): while a stage is multiplied
// the next one is on its way, with one barrier a stage. An operand whose memory runs along k lies in rows of 64 k (128 bytes), its 16-byte
// chunks exchanged by the row's low bits, so that the reads of eight rows meet all banks; one whose memory runs along i (or j) lies as it
// is, 256 (128) to a row of k, and is read by the transposing read, four rows of k by 16 columns to 16 lanes, its pairs of chunks
// exchanged by k's bits. What lies past an operand's end is read as zero by the buffer's bounds.
//
// A lane's results are four consecutive i at one j: in the logits i is the table row, so that a row's maximum and sum
// stay mostly in registers; the gradients are stored along i.
//
// The matrix unit bounds it, and its power: the four products of 8,192 x 128,000 x 4,096 bfloat16 run at 1,235 TFLOP/s (logits 6.6 ms, the gradients' 7.1, 6.8
// and 7.3 in eight pieces) at 1.8 GHz with the unit busy for 65 % of the cycles; a library's product of the same operands reaches 1,270 at 1.46 GHz and 83 %.
// What led there, in ms of the logits: every transfer and read ahead of a step's products 7.16, the next half step's reads between them 6.94, its transfers too
// 6.73. v_mfma_f32_32x32x16 instead: 7.02. 2,047 x 49,999 x 1,024: logits 241 us, gradients 264, 191 and 278 (196 x 8 tiles are 6.1 rounds of the 256 CUs and
// take seven). 1,001 x 10,007 x 333 float16: 19, 25, 20 and 23 us, the last two by small tiles (with large ones the pass takes 127 us instead of 111).
// Floats, 8,192 x 32,000 x 4,096: 41.3 ms a pass, 68.0 on the float32 instruction (126 TFLOP/s); 2,047 x 49,999 x 1,024: 5.1 and 7.2, the features' gradient
// 4e-8 and 1.4e-6 off.
#include <algorithm>
#include <type_traits>

#include "cross_entropy.h"

namespace efgs {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef short shortx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

constexpr uint32_t step_k = 64, wave_chunks = 4;                // transfers of 1 KB by a wave to an operand's tile
template <uint32_t SIDE> constexpr uint32_t block_of = SIDE * 2;
template <typename T> constexpr uint32_t parts_of = std::is_same_v<T, float> ? 3 : 1;   // a float: bfloat16 parts
template <typename T> using Element = std::conditional_t<std::is_same_v<T, float>, __bf16, T>;
constexpr uint32_t pairs = 6;                                   // of parts, the smallest products first; those below 2^-24 of the largest are left out
__device__ __forceinline__ uint32_t a_part(uint32_t pair) { return 0x001012u >> 4 * pair & 3u; }
__device__ __forceinline__ uint32_t b_part(uint32_t pair) { return 0x010210u >> 4 * pair & 3u; }
constexpr uint32_t outside = 0xfffffff0u;                       // an offset past every bound
constexpr float infinity = __builtin_inff();

// a product that is rounded before it is subtracted from, as the forward has it
__device__ __forceinline__ float rounded(float x) {
    asm("" : "+v"(x));
    return x;
}

template <typename T>
__device__ __forceinline__ floatx4 multiply(shortx8 a, shortx8 b, floatx4 c) {
    if constexpr (std::is_same_v<T, __bf16>) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, a), __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
}

// 64 lanes' 16 bytes each to 1 KB of LDS at `to`. (The builtin of this transfer makes the compiler wait for it before the next
// transposing read of whatever address; the waits stand in the loop instead.)
__device__ __forceinline__ void to_lds(uint32_t to, uintx4 buffer, uint32_t lane_offset, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(lane_offset), "s"(buffer), "s"(offset) : "memory", "m0");
}

__device__ __forceinline__ uint32_t scalar(uint32_t x) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))); }

__device__ __forceinline__ uintx4 buffer_of(const void* base, uint64_t bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    return uintx4{scalar(static_cast<uint32_t>(at)), scalar(static_cast<uint32_t>(at >> 32)), scalar(bytes < 0xffffff00u ? static_cast<uint32_t>(bytes) : 0xffffff00u),
                  0x00020000u};
}

// An operand: ALONG_K, `first` its first row of the tile (of `rows`), k along them; otherwise `first` the tile's first column, k the row.
template <uint32_t SIDE, bool ALONG_K>
struct Operand {
    const char* base;
    uint64_t stride;         // bytes
    uint32_t rows, columns;  // as they lie in memory
    uint32_t first, k_end;
    uintx4 buffer;
    uint32_t offsets[wave_chunks];
    uint32_t chunk_k;        // ALONG_K: k of the lane's 16 bytes within a step

    __device__ __forceinline__ void begin(const void* p, uint64_t stride_elements, uint32_t rows_, uint32_t columns_, uint32_t first_, uint32_t k_end_) {
        const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
        base = static_cast<const char*>(p);
        stride = stride_elements * 2;
        rows = rows_;
        columns = columns_;
        first = first_;
        k_end = k_end_;
        if constexpr (ALONG_K) {
            const uint64_t left = min(rows - first, SIDE);
            buffer = buffer_of(base + first * stride, (left - 1) * stride + columns * 2ull);
            chunk_k = ((lane & 7u) ^ (lane >> 3)) * 8;
#pragma unroll
            for (uint32_t u = 0; u < wave_chunks; u++)
                offsets[u] = ((wave * wave_chunks + u) * 8 + (lane >> 3)) * static_cast<uint32_t>(stride) + chunk_k * 2;
        } else {
#pragma unroll
            for (uint32_t u = 0; u < wave_chunks; u++) {
                constexpr uint32_t lanes = SIDE / 8;  // of a row
                const uint32_t k = (wave * wave_chunks + u) * (64 / lanes) + lane / lanes, exchange = (k & 3u) | (k >> 3 & 1u) << 2;
                offsets[u] = k * static_cast<uint32_t>(stride) + (first + (lane % lanes ^ 2 * exchange) * 8) * 2;
            }
        }
    }

    // transfer u of the tile of k..k + 63, `part` elements on, which `buffer_at` describes, on its way to LDS at `to` (past k's end: zeros)
    __device__ __forceinline__ uintx4 buffer_at(uint32_t k, uint32_t part) const {
        if constexpr (ALONG_K) return buffer;
        const uint64_t left = min(k_end - min(k, k_end), step_k);
        return buffer_of(base + k * stride + part * 2ull, left > 0 ? (left - 1) * stride + columns * 2ull : 0);
    }

    __device__ __forceinline__ void load(uint32_t to, uintx4 here, uint32_t k, uint32_t part, uint32_t u) const {
        const uint32_t at = to + (scalar(threadIdx.x >> 6) * wave_chunks + u) * 1024;
        if constexpr (ALONG_K) to_lds(at, here, k + chunk_k < k_end ? offsets[u] : outside, k < k_end ? (part + k) * 2 : 0);
        else to_lds(at, here, offsets[u], 0);
    }
};

// Fragments of a step: lane (e, q) holds k = 8 q..8 q + 7 of each half step of 32 at column e of each 16.
template <uint32_t SIDE, bool ALONG_K, uint32_t N>
struct Fragments {
    static constexpr uint32_t row_bytes = SIDE * 2;  // of k
    uint32_t at[ALONG_K ? 2 : N];

    __device__ __forceinline__ void begin(uint32_t first) {
        const uint32_t lane = threadIdx.x & 63u, e = lane & 15u, q = lane >> 4;
        if constexpr (ALONG_K) {
#pragma unroll
            for (uint32_t half = 0; half < 2; half++) at[half] = (first + e) * 128 + ((half * 4 + q) ^ (e & 7u)) * 16;
        } else {
            const uint32_t exchange = (e >> 2) | (q & 1u) << 2;
#pragma unroll
            for (uint32_t t = 0; t < N; t++) at[t] = (8 * q + (e >> 2)) * row_bytes + ((first / 16 + t) ^ exchange) * 32 + (e & 3u) * 8;
        }
    }

    __device__ __forceinline__ shortx8 read(const char* lds, uint32_t half, uint32_t t) const {
        if constexpr (ALONG_K) {
            return *reinterpret_cast<const shortx8*>(lds + at[half] + t * 2048);
        } else {
            using Part = __attribute__((address_space(3))) shortx4;
            const shortx4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Part*)(lds + at[t] + half * 32 * row_bytes));
            const shortx4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Part*)(lds + at[t] + (half * 32 + 4) * row_bytes));
            return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// The logits' gradients are rounded to the type. A row's own target's is mostly the largest by far, and its rounding would be most of what the gradients lose;
// so what it lost is added to them, in the rows' gradient as they are gathered, and in the table's here: the packed rows of the block's share of k whose target is
// one of the tile's table rows are looked up, and 64 of them at a time make one more step of k, their features one operand and the residuals, each in its
// row and target's column of zeros, the other; the next 64 rows' features are on their way meanwhile. (8,192 rows against 128,000: sixteen of them to a tile,
// mostly one step after 128.) A float's target's gradient is left out of the piece as a whole and added here, by its parts: a sum over a long table that holds
// one large value from early on rounds all that follow to it.
template <typename T, uint32_t SIDE, typename FA, typename FB, typename Acc>
__device__ __forceinline__ void add_residuals(const EntropyProductArgs& a, char* lds, uint32_t begin, uint32_t end, uint32_t i0, uint32_t j0, const FA& fragments_a,
                                              const FB& fragments_b, Acc& acc) {
    constexpr uint32_t block = block_of<SIDE>, operand_bytes = SIDE * step_k * 2, row_bytes = SIDE * 2, at_once = 4, most = SIDE * 32;
    constexpr uint32_t wave_i = SIDE / 32, wave_j = 4, parts = parts_of<T>, chunks = operand_bytes / 16 / block;   // of 16 bytes, of an operand
    using E = Element<T>;
    uint32_t* const list = reinterpret_cast<uint32_t*>(lds + 2 * operand_bytes);   // the second stage: packed rows, then the waves' counts
    uint32_t* const wave_counts = list + most;
    static_assert((most + at_once * block / 64) * sizeof(uint32_t) <= 2 * operand_bytes, "the list fits a stage");
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, first = a.first_row + j0;
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    uint32_t listed = 0;
    E* place = reinterpret_cast<E*>(lds + operand_bytes);   // of the thread's row's residual
    __syncthreads();
#pragma unroll
    for (uint32_t c = 0; c < chunks; c++) *reinterpret_cast<Words*>(lds + operand_bytes + (c * block + threadIdx.x) * 16) = Words{};
    for (uint32_t from = begin; from < end; from += at_once * block) {
        bool hit[at_once];
#pragma unroll
        for (uint32_t k = 0; k < at_once; k++) {
            const uint32_t m = from + k * block + threadIdx.x;
            hit[k] = m < end && a.target[m] - first < SIDE;
        }
#pragma unroll
        for (uint32_t k = 0; k < at_once; k++) {
            const uint64_t ballot = __ballot(hit[k]);
            if (lane == 0) wave_counts[k * (block / 64) + wave] = static_cast<uint32_t>(__popcll(ballot));
        }
        __syncthreads();
        uint32_t before[at_once] = {}, all = 0;
        for (uint32_t w = 0; w < at_once * block / 64; w++) {
            const uint32_t n = wave_counts[w];
#pragma unroll
            for (uint32_t k = 0; k < at_once; k++) before[k] += w < k * (block / 64) + wave ? n : 0u;
            all += n;
        }
#pragma unroll
        for (uint32_t k = 0; k < at_once; k++) {
            const uint64_t ballot = __ballot(hit[k]);
            if (hit[k]) list[listed + before[k] + static_cast<uint32_t>(__popcll(ballot & ((1ull << lane) - 1ull)))] = from + k * block + threadIdx.x;
        }
        listed += all;
        __syncthreads();
        if (listed == 0 || (from + at_once * block < end && listed + at_once * block <= most)) continue;
        Words next[chunks];
        float next_residual = 0.0f;
        uint32_t next_column = 0;   // of the tile: the target's
        const auto fetch = [&](uint32_t k0, uint32_t part) {
#pragma unroll
            for (uint32_t c = 0; c < chunks; c++) {
                const uint32_t at = c * block + threadIdx.x, k = at / (row_bytes / 16), chunk = at % (row_bytes / 16), exchange = (k & 3u) | (k >> 3 & 1u) << 2;
                const uint32_t column = i0 + (chunk ^ 2 * exchange) * 8;
                next[c] = Words{};
                if (k0 + k < listed && column < a.a_columns)
                    next[c] = *reinterpret_cast<const Words*>(static_cast<const E*>(a.a) + list[k0 + k] * a.a_stride + part * a.a_plane + column);
            }
            if (threadIdx.x < step_k) {
                const bool inside = k0 + threadIdx.x < listed;
                const uint32_t m = inside ? list[k0 + threadIdx.x] : 0;
                next_residual = inside ? a.residual[m] : 0.0f;
                next_column = inside ? a.target[m] - first : 0;
            }
        };
        fetch(0, 0);
        for (uint32_t k0 = 0; k0 < listed; k0 += step_k) {
            for (uint32_t part = 0; part < parts; part++) {
                float left = next_residual;
#pragma unroll
                for (uint32_t c = 0; c < chunks; c++) *reinterpret_cast<Words*>(lds + (c * block + threadIdx.x) * 16) = next[c];
                if (threadIdx.x < step_k) {
                    const uint32_t k = threadIdx.x, v = next_column, exchange = (k & 3u) | (k >> 3 & 1u) << 2;
                    *place = static_cast<E>(0.0f);
                    place = reinterpret_cast<E*>(lds + operand_bytes + k * row_bytes + (v / 16 ^ exchange) * 32 + v % 16 * 2);
                }
                for (uint32_t other = 0; other < parts - part; other++) {  // the residual's parts that go with this one of the features
                    if (other > 0) __syncthreads();
                    if (threadIdx.x < step_k) *place = static_cast<E>(left);
                    left -= static_cast<float>(static_cast<E>(left));
                    __syncthreads();
                    if (other == 0) fetch(part + 1 < parts ? k0 : k0 + step_k, part + 1 < parts ? part + 1 : 0);
#pragma unroll
                    for (uint32_t half = 0; half < 2; half++) {
                        shortx8 fa[wave_i], fb[wave_j];
#pragma unroll
                        for (uint32_t t = 0; t < wave_j; t++) fb[t] = fragments_b.read(lds + operand_bytes, half, t);
#pragma unroll
                        for (uint32_t t = 0; t < wave_i; t++) fa[t] = fragments_a.read(lds, half, t);
#pragma unroll
                        for (uint32_t ti = 0; ti < wave_i; ti++)
#pragma unroll
                            for (uint32_t tj = 0; tj < wave_j; tj++) acc[ti][tj] = multiply<E>(fa[ti], fb[tj], acc[ti][tj]);
                    }
                }
                __syncthreads();
            }
        }
        listed = 0;
    }
}

// A step of k; of floats, the steps of one pair of parts follow those of another.
template <uint32_t PARTS>
struct Step {
    uint32_t k, first, end, a_plane, b_plane, pair;

    __device__ __forceinline__ void advance() {
        k += step_k;
        if constexpr (PARTS == 3) {
            if (k >= end) {
                pair++;
                k = pair < pairs ? first : end;
            }
        }
    }
    __device__ __forceinline__ uint32_t of_a() const { return PARTS == 3 ? a_part(pair) * a_plane : 0; }
    __device__ __forceinline__ uint32_t of_b() const { return PARTS == 3 ? b_part(pair) * b_plane : 0; }
};

template <typename T, EntropyProduct P, uint32_t SIDE>
__global__ __launch_bounds__(block_of<SIDE>, 2) void entropy_wide_kernel(EntropyProductArgs a) {
    constexpr bool first_two = P == entropy_logits || P == entropy_upstream, a_along_k = first_two, b_along_k = P != entropy_table_gradient;
    constexpr uint32_t tile = SIDE, operand_bytes = tile * step_k * 2, stage_bytes = 2 * operand_bytes;
    constexpr uint32_t wave_i = SIDE / 32, wave_j = 4;  // tiles of 16 a wave
    constexpr uint32_t parts = parts_of<T>;
    using E = Element<T>;
    __shared__ __attribute__((aligned(1024))) char lds[2 * stage_bytes];
    const uint32_t count = scalar(*a.count);
    // Blocks go round the eight XCDs one by one: each XCD takes a run of the tiles, split by split, four rows of j at a time along i, so that the tiles
    // that are under way on it share their operands in its L2.
    const uint32_t j_tiles = P == entropy_table_gradient ? (a.j_end + tile - 1) / tile
                                                         : (min(count - min(count, a.j_first), a.j_end) + tile - 1) / tile;
    const uint32_t tiles = a.i_tiles * j_tiles, blocks = tiles * a.splits, each = (blocks + 7) / 8, in_all = (blockIdx.x & 7u) * each + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= each || in_all >= blocks) return;
    const uint32_t split = in_all / tiles, at = in_all - split * tiles;
    const uint32_t band = at / (4 * a.i_tiles), in_band = at - band * 4 * a.i_tiles, width = min(4u, j_tiles - band * 4);
    const uint32_t i0 = in_band / width * tile, j0 = a.j_first + (band * 4 + in_band % width) * tile;
    const uint32_t k_all = P == entropy_table_gradient ? (count + step_k - 1) / step_k * step_k : a.k_end;
    const uint32_t k_each = ((k_all + a.splits - 1) / a.splits + step_k - 1) / step_k * step_k;
    const uint32_t k_first = min(split * k_each, k_all), k_end = min(k_first + k_each, k_all);

    const uint32_t lane = threadIdx.x & 63u, e = lane & 15u, q = lane >> 4, wave = threadIdx.x >> 6, wi = wave & 1u, wj = wave >> 1;
    const uint32_t b_columns = parts > 1 ? a.b_plane : static_cast<uint32_t>(a.b_stride);  // of a part
    Operand<SIDE, a_along_k> operand_a;
    Operand<SIDE, b_along_k> operand_b;
    if constexpr (first_two) {
        operand_a.begin(a.a, a.a_stride, a.i_end, a.a_columns, i0, parts > 1 ? a.a_plane : a.a_columns);
        operand_b.begin(a.b, a.b_stride, j0 + tile, static_cast<uint32_t>(a.b_stride), j0, b_columns);
    } else if constexpr (P == entropy_features_gradient) {
        operand_a.begin(a.a, a.a_stride, k_all, a.a_columns, i0, k_all);
        operand_b.begin(a.b, a.b_stride, j0 + tile, static_cast<uint32_t>(a.b_stride), j0, b_columns);
    } else {
        operand_a.begin(a.a, a.a_stride, k_all, a.a_columns, i0, k_all);
        operand_b.begin(a.b, a.b_stride, k_all, b_columns, j0, k_all);
    }
    Fragments<SIDE, a_along_k, wave_i> fragments_a;
    Fragments<SIDE, b_along_k, wave_j> fragments_b;
    fragments_a.begin(wi * (SIDE / 2));
    fragments_b.begin(wj * 64);
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<uint64_t>((__attribute__((address_space(3))) char*)lds));

    floatx4 acc[wave_i][wave_j] = {};
    shortx8 fa[2][wave_i], fb[2][wave_j];  // of the two halves of a step
    // A half step: its products, and between them, so that both are under way at once, the reads of the fragments of the half step behind it
    // and, in the second half, the transfers of the step after the next.
    const auto half_step = [&](auto half, const char* from, uint32_t to, const Step<parts>& s) {
        constexpr uint32_t h = decltype(half)::value;
        uintx4 buffer_a{}, buffer_b{};
        if constexpr (h == 1) {
            buffer_a = operand_a.buffer_at(s.k, s.of_a());
            buffer_b = operand_b.buffer_at(s.k, s.of_b());
        }
#pragma unroll
        for (uint32_t ti = 0; ti < wave_i; ti++) {
            if (ti < wave_j) fb[1 - h][ti] = fragments_b.read(from + operand_bytes, 1 - h, ti);
            fa[1 - h][ti] = fragments_a.read(from, 1 - h, ti);
            if (h == 1 && ti < wave_chunks) {
                operand_a.load(to, buffer_a, s.k, s.of_a(), ti);
                operand_b.load(to + operand_bytes, buffer_b, s.k, s.of_b(), ti);
            }
#pragma unroll
            for (uint32_t tj = 0; tj < wave_j; tj++) acc[ti][tj] = multiply<E>(fa[h][ti], fb[h][tj], acc[ti][tj]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const std::integral_constant<uint32_t, 0> first_half;
    const std::integral_constant<uint32_t, 1> second_half;
    // (Steps past the end are read as zeros, so that nothing stands in branches.) Half way through a step its second half is in the registers: its
    // stage is free for the step after the next, and the next one's has to be there.
    if (k_first < k_end) {
        Step<parts> ahead{k_first, k_first, k_end, a.a_plane, a.b_plane, 0};
        const auto load = [&](uint32_t to) {
            const uintx4 buffer_a = operand_a.buffer_at(ahead.k, ahead.of_a()), buffer_b = operand_b.buffer_at(ahead.k, ahead.of_b());
#pragma unroll
            for (uint32_t u = 0; u < wave_chunks; u++) {
                operand_a.load(to, buffer_a, ahead.k, ahead.of_a(), u);
                operand_b.load(to + operand_bytes, buffer_b, ahead.k, ahead.of_b(), u);
            }
            ahead.advance();
        };
        load(lds_at);
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        load(lds_at + stage_bytes);
#pragma unroll
        for (uint32_t t = 0; t < wave_j; t++) fb[0][t] = fragments_b.read(lds + operand_bytes, 0, t);
#pragma unroll
        for (uint32_t t = 0; t < wave_i; t++) fa[0][t] = fragments_a.read(lds, 0, t);
        uint32_t stage = 0;
        for (uint32_t n = (k_end - k_first + step_k - 1) / step_k * (parts > 1 ? pairs : 1); n > 0; n--) {
            half_step(first_half, lds + stage, 0, ahead);
            __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0): this wave's part of the next stage is there, its reads of this one are done
            __builtin_amdgcn_s_barrier();        // and so for the other waves
            asm volatile("" ::: "memory");
            half_step(second_half, lds + (stage ^ stage_bytes), lds_at + stage, ahead);
            ahead.advance();
            stage ^= stage_bytes;
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the zeros that follow the last step
    }

    if constexpr (P == entropy_table_gradient) {
        if (a.apart) add_residuals<T, SIDE>(a, lds, k_first, min(k_end, count), i0, j0, fragments_a, fragments_b, acc);
    }
    const uint32_t i_lane = i0 + wi * (SIDE / 2) + 4 * q, j_lane = j0 + wj * 64 + e;  // results: i_lane + 16 ti + r, j_lane + 16 tj
    if constexpr (P == entropy_logits) {
        __syncthreads();
        float2* const joined = reinterpret_cast<float2*>(lds);
#pragma unroll
        for (uint32_t tj = 0; tj < wave_j; tj++) {
            const uint32_t j = j_lane + tj * 16, target = a.target[j];
            float top = -infinity, sum = 0.0f;
#pragma unroll
            for (uint32_t ti = 0; ti < wave_i; ti++)
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) {
                    const uint32_t i = i_lane + ti * 16 + r;
                    const float z = i < a.i_end ? acc[ti][tj][r] * a.to_log2 : -infinity;
                    acc[ti][tj][r] = z;
                    if (i == target) a.target_logit[j] = z;
                    top = fmaxf(top, z);
                }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float from = top == -infinity ? 0.0f : top;
#pragma unroll
            for (uint32_t ti = 0; ti < wave_i; ti++)
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) sum += __builtin_amdgcn_exp2f(acc[ti][tj][r] - from);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (q == 0) joined[wi * tile + wj * 64 + tj * 16 + e] = make_float2(top, sum);
        }
        __syncthreads();
        if (threadIdx.x < tile) {
            const float2 x = joined[threadIdx.x], y = joined[tile + threadIdx.x];
            const float top = fmaxf(x.x, y.x), from = top == -infinity ? 0.0f : top;
            const float sum = x.y * __builtin_amdgcn_exp2f(x.x - from) + y.y * __builtin_amdgcn_exp2f(y.x - from);
            a.partial[(i0 / tile) * a.slab_rows + (j0 - a.j_first) + threadIdx.x] = make_float2(top, sum);
        }
    } else if constexpr (P == entropy_upstream) {
        typedef E Four __attribute__((ext_vector_type(4)));
#pragma unroll
        for (uint32_t tj = 0; tj < wave_j; tj++) {
            const uint32_t j = j_lane + tj * 16, target = a.target[j];
            const bool counts = target != entropy_none;
            const float2 lse = counts ? a.lse[j] : make_float2(0.0f, 0.0f);
            const float weight = counts ? a.weight[j] : 0.0f;
            const bool hit = __any(target - (a.first_row + i0 + wi * (SIDE / 2)) < SIDE / 2);  // a target among the wave's table rows
#pragma unroll
            for (uint32_t ti = 0; ti < wave_i; ti++) {
                const uint32_t i = i_lane + ti * 16;
                floatx4 p;
                E* const piece = static_cast<E*>(a.piece) + j * a.piece_stride + i;
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) p[r] = __builtin_amdgcn_exp2f((rounded(acc[ti][tj][r] * a.to_log2) - lse.x) - lse.y);
                if (hit) {
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++)
                        if (a.first_row + i + r == target) p[r] -= 1.0f;
                }
                if constexpr (parts == 1) {
                    Four g;
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) g[r] = static_cast<T>(counts && i + r < a.i_end ? p[r] * weight : 0.0f);
                    if (hit) {
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++)
                            if (a.first_row + i + r == target) a.residual[j] = p[r] * weight - static_cast<float>(g[r]);
                    }
                    *reinterpret_cast<Four*>(piece) = g;
                } else {
                    float g[4];
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) {
                        g[r] = counts && i + r < a.i_end ? p[r] * weight : 0.0f;
                        if (hit && a.apart && a.first_row + i + r == target) {
                            a.residual[j] = g[r];
                            g[r] = 0.0f;
                        }
                    }
                    Four split[parts];
                    entropy_split<parts>(split, g);
#pragma unroll
                    for (uint32_t part = 0; part < parts; part++) *reinterpret_cast<Four*>(piece + part * a.piece_plane) = split[part];
                }
            }
        }
    } else {
        typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
        const bool direct = P == entropy_table_gradient && a.out;
        const float factor = direct ? *a.factor : 1.0f;
        const uint32_t j_end = P == entropy_table_gradient ? a.j_end : count;
#pragma unroll
        for (uint32_t tj = 0; tj < wave_j; tj++) {
            const uint32_t j = j_lane + tj * 16;
            if (j >= j_end) continue;
#pragma unroll
            for (uint32_t ti = 0; ti < wave_i; ti++) {
                const uint32_t i = i_lane + ti * 16;
                if (direct) {
                    T* const out = static_cast<T*>(a.out) + j * a.out_stride + i;
                    Four y;
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) y[r] = static_cast<T>(acc[ti][tj][r] * factor);
                    if (i + 4 <= a.i_end) *reinterpret_cast<Four*>(out) = y;
                    else
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++)
                            if (i + r < a.i_end) out[r] = y[r];
                } else if (i < a.slab_stride) {
                    floatx4* const out = reinterpret_cast<floatx4*>(a.slab + (split * a.slab_rows + j) * a.slab_stride + i);
                    *out = a.add ? *out + acc[ti][tj] : acc[ti][tj];
                }
            }
        }
    }
}

template <typename T, uint32_t SIDE>
void launch(EntropyProduct product, const EntropyProductArgs& a, uint32_t j, hipStream_t s) {
    const dim3 grid((a.i_tiles * div_up(j, SIDE) * a.splits + 7) / 8 * 8), block(block_of<SIDE>);
    switch (product) {
        case entropy_logits: hipLaunchKernelGGL((entropy_wide_kernel<T, entropy_logits, SIDE>), grid, block, 0, s, a); break;
        case entropy_upstream: hipLaunchKernelGGL((entropy_wide_kernel<T, entropy_upstream, SIDE>), grid, block, 0, s, a); break;
        case entropy_features_gradient: hipLaunchKernelGGL((entropy_wide_kernel<T, entropy_features_gradient, SIDE>), grid, block, 0, s, a); break;
        case entropy_table_gradient: hipLaunchKernelGGL((entropy_wide_kernel<T, entropy_table_gradient, SIDE>), grid, block, 0, s, a); break;
    }
}

}  // namespace

void launch_entropy_wide(EntropyProduct product, int type, uint32_t side, const EntropyProductArgs& a, uint32_t j, hipStream_t s) {
    if (type == type_bfloat16) {
        if (side == 256) launch<__bf16, 256>(product, a, j, s);
        else launch<__bf16, 128>(product, a, j, s);
    } else if (type == type_half) {
        if (side == 256) launch<_Float16, 256>(product, a, j, s);
        else launch<_Float16, 128>(product, a, j, s);
    } else {
        if (side == 256) launch<float, 256>(product, a, j, s);
        else launch<float, 128>(product, a, j, s);
    }
}

}  // namespace efgs
