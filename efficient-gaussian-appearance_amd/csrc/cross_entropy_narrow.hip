// The cross entropy for rows of few columns (codes): the logits of a tile of both sides never leave the registers.
//
// A wave owns up to 64 rows of one side, 16 to a tile, and meets the rows of the other side 16 at a time, from LDS:
//   logits      S(m, o) = sum_k stream(m, k) own(o, k)        a lane has four m at one o
//   gradient    out(d, o) += sum_m stream(m, d) g(m, o)       g's registers as they lie are this product's operand: register r of lane (o, q) is row 4 q + r
// The forward and the rows' gradient own packed rows and meet the table; the table's gradient owns table rows and meets the packed rows. Sums that
// several blocks or waves share are left as partial ones, joined in their order.
//
// All products are v_mfma_f32_16x16x32_bf16 of parts: a float is the sum of three bfloat16 to 2^-26 of it (a float16 of two, exactly), and the parts'
// products below 2^-24 of the largest are left out, so that nothing is lost against float32 products. Those, on v_mfma_f32_16x16x4_f32, take the vector
// unit's time beside its own (counted: 54 % and 46 % of a gradient kernel's cycles) where these run beside it. A step of
// k = 32 is four slots of eight, one to each quarter of the wave: the columns of a block of eight times one pair of parts; in
// the gradient a lane's four rows times two parts of g.
//
// 1,000,000 x 4,096 x 8 float32: logits 1.09 ms, the features' gradient 1.77, the table's 1.88. The vector unit bounds them: 4.1 G exponentials in each at a
// quarter of its rate are 0.4 ms by themselves, and the gradients split every g in three parts (15 operations for two of them). By v_mfma_f32_16x16x4_f32
// 1.27, 2.25 and 2.23; with the logits' gradients in memory 40 ms a pass. 32,768 x 4,096 x 64 float32: 0.12, 0.20 and 0.20 ms.
#include <algorithm>
#include <type_traits>

#include "cross_entropy.h"

namespace efgs {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t block = 256, waves = 4, chunk = 64, chunk_tiles = chunk / 16;
constexpr float infinity = __builtin_inff();
constexpr float far_above = 64.0f;   // how far (log 2) a logit may lie above the lane's reference: what sums of 2^64 and below leave room for

__device__ __forceinline__ uint32_t scalar(uint32_t x) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))); }

// bfloat16 parts of a value, and the slots of a block of eight columns: pairs of parts (stream's, own's)
template <typename T> constexpr uint32_t parts_of = std::is_same_v<T, float> ? 3 : std::is_same_v<T, __bf16> ? 1 : 2;
template <uint32_t PARTS> constexpr uint32_t slots_of = PARTS == 3 ? 6 : PARTS == 2 ? 4 : 1;
template <uint32_t PARTS> __device__ __forceinline__ uint32_t stream_part(uint32_t pair) { return PARTS == 1 ? 0 : PARTS == 2 ? pair >> 1 : 0x120100u >> 4 * pair & 3u; }
template <uint32_t PARTS> __device__ __forceinline__ uint32_t own_part(uint32_t pair) { return PARTS == 1 ? 0 : PARTS == 2 ? pair & 1u : 0x102010u >> 4 * pair & 3u; }

__device__ __forceinline__ floatx4 multiply(bf16x8 a, bf16x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ bf16x8 pair(bf16x4 a, bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

// KB: blocks of eight columns; TILES: of 16 owned rows a wave
// (two blocks to a CU: half of the registers, so that products stay in those the vector unit reads)
template <typename T, EntropyProduct P, int KB, int TILES>
__global__ __launch_bounds__(block, 2) void entropy_narrow_kernel(EntropyNarrowArgs a) {
    constexpr bool gradient = P != entropy_logits, own_table = P == entropy_table_gradient;
    constexpr uint32_t PARTS = parts_of<T>, SLOTS = slots_of<PARTS>, MS = (KB * SLOTS + 3) / 4, DT = (KB + 1) / 2;
    // steps after which the slots come again, and their column blocks
    constexpr uint32_t period = PARTS == 3 ? 3 : 1, period_blocks = PARTS == 3 ? 2 : PARTS == 2 ? 1 : 4;
    constexpr uint32_t part_bytes = KB * chunk * 16;
    __shared__ __attribute__((aligned(16))) char lds[PARTS * part_bytes];                  // part, column block, row: eight columns
    // of the streamed rows: the log sum's first part; the weight times what the second makes of a probability; the weight
    __shared__ __attribute__((aligned(16))) float row_first[own_table ? chunk : 4], row_factor[own_table ? chunk : 4], row_weight[own_table ? chunk : 4];
    __shared__ __attribute__((aligned(16))) uint32_t row_target[own_table ? chunk : 4];
    const uint32_t count = scalar(*a.count), own_end = own_table ? a.table_rows : count, stream_end = own_table ? count : a.table_rows;
    const uint32_t lane = threadIdx.x & 63u, e = lane & 15u, q = lane >> 4, wave = scalar(threadIdx.x >> 6);
    const uint32_t stream_waves = waves / a.own_waves, own_wave = wave / stream_waves, stream_wave = wave % stream_waves;
    const uint32_t own_first = (blockIdx.x * a.own_waves + own_wave) * TILES * 16;
    if (blockIdx.x * a.own_waves * TILES * 16 >= own_end) return;
    const uint32_t chunks = (stream_end + chunk - 1) / chunk, chunks_each = (chunks + gridDim.y - 1) / gridDim.y;
    const uint32_t begin = min(blockIdx.y * chunks_each, chunks) * chunk, end = min(stream_end, begin + chunks_each * chunk);
    const T* const own = static_cast<const T*>(own_table ? a.table : a.packed);
    const T* const stream = static_cast<const T*>(own_table ? a.packed : a.table);
    const uint64_t own_stride = own_table ? a.table_stride : a.packed_stride, stream_stride = own_table ? a.packed_stride : a.table_stride;

    bf16x8 fo[TILES][MS];
    float own_lse[TILES], own_one[TILES], own_factor[TILES];  // the log sum's first part; what the second makes of 1, and its reciprocal
    uint32_t target[TILES];
    floatx4 out[TILES][DT];
    float reference[TILES], sum[TILES];
    bool begun[TILES];
#pragma unroll
    for (uint32_t t = 0; t < TILES; t++) {
        const uint32_t o = own_first + t * 16 + e;
        const bool inside = o < own_end;
#pragma unroll
        for (uint32_t s = 0; s < MS; s++) {
            const uint32_t slot = 4 * s + q, column = slot / SLOTS * 8, part = own_part<PARTS>(slot % SLOTS);
            float x[8];
            entropy_load8<T>(x, own + o * own_stride + column, inside && slot < KB * SLOTS ? static_cast<int32_t>(a.columns) - static_cast<int32_t>(column) : 0);
            bf16x8 parts[PARTS];
            entropy_split<PARTS>(parts, x);
            fo[t][s] = parts[0];
#pragma unroll
            for (uint32_t k = 1; k < PARTS; k++) fo[t][s] = part == k ? parts[k] : fo[t][s];
        }
        const float2 lse = P == entropy_features_gradient && inside ? a.lse[o] : make_float2(0.0f, 0.0f);
        own_lse[t] = lse.x;
        own_one[t] = __builtin_amdgcn_exp2f(lse.y);
        own_factor[t] = __builtin_amdgcn_exp2f(-lse.y);
        target[t] = !own_table && inside ? a.target[o] : entropy_none;
        reference[t] = 0.0f;
        begun[t] = false;
        sum[t] = 0.0f;
#pragma unroll
        for (uint32_t d = 0; d < DT; d++) out[t][d] = floatx4{};
    }
    // where the lane's rows and columns of the streamed tile lie
    uint32_t row_at[period], column_at[DT];
#pragma unroll
    for (uint32_t s = 0; s < period; s++) {
        const uint32_t slot = 4 * s + q;
        row_at[s] = stream_part<PARTS>(slot % SLOTS) * part_bytes + (min(slot / SLOTS, KB - 1u) * chunk + e) * 16;
    }
#pragma unroll
    for (uint32_t d = 0; d < DT; d++) column_at[d] = (min(2 * d + (e >> 1 & 1u), KB - 1u) * chunk + 4 * q + (e >> 2)) * 16 + (e & 1u) * 8;

    // a chunk of the streamed rows on its way to the registers: row threadIdx.x / 4, every fourth block of its columns
    constexpr uint32_t blocks = (KB + 3) / 4;
    const uint32_t row = threadIdx.x / 4, first_block = threadIdx.x % 4;
    float next[blocks][8];
    float2 next_lse{};
    float next_weight = 0.0f;
    uint32_t next_target = entropy_none;
    const auto fetch = [&](uint32_t from) {
        const uint32_t m = from + row;
#pragma unroll
        for (uint32_t j = 0; j < blocks; j++) {
            const uint32_t column = (first_block + 4 * j) * 8;
            entropy_load8<T>(next[j], stream + static_cast<uint64_t>(m) * stream_stride + column,
                     m < stream_end ? static_cast<int32_t>(a.columns) - static_cast<int32_t>(column) : 0);
        }
        if constexpr (own_table) {
            next_lse = m < stream_end ? a.lse[m] : make_float2(infinity, 0.0f);  // (no probability)
            next_weight = m < stream_end ? a.weight[m] : 0.0f;
            next_target = m < stream_end ? a.target[m] : entropy_none;
        }
    };
    if (begin < end) fetch(begin);
    for (uint32_t from = begin; from < end; from += chunk) {
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < blocks; j++) {
            const uint32_t b = first_block + 4 * j;
            if (b < KB) {
                bf16x8 parts[PARTS];
                entropy_split<PARTS>(parts, next[j]);
#pragma unroll
                for (uint32_t part = 0; part < PARTS; part++) *reinterpret_cast<bf16x8*>(lds + part * part_bytes + (b * chunk + row) * 16) = parts[part];
            }
        }
        if constexpr (own_table) {
            if (first_block == 0) {
                row_first[row] = next_lse.x;
                row_factor[row] = __builtin_amdgcn_exp2f(-next_lse.y) * next_weight;
                row_weight[row] = next_weight;
                row_target[row] = next_target;
            }
        }
        __syncthreads();
        if (from + chunk < end) fetch(from + chunk);
        for (uint32_t mt = stream_wave; mt < chunk_tiles; mt += stream_waves) {
            const uint32_t m0 = from + mt * 16;
            if (m0 >= end) break;
            floatx4 z[TILES];
#pragma unroll
            for (uint32_t t = 0; t < TILES; t++) z[t] = floatx4{};
#pragma unroll
            for (uint32_t s = 0; s < MS; s++) {
                const uint32_t at = PARTS == 1 ? (min(4 * s + q, KB - 1u) * chunk + e) * 16 : row_at[s % period] + s / period * period_blocks * chunk * 16;
                const bf16x8 fs = *reinterpret_cast<const bf16x8*>(lds + at + mt * 256);
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++) z[t] = multiply(fs, fo[t][s], z[t]);
            }
            if constexpr (!gradient) {
                bool above = false;
                float top[TILES];  // above the reference, or the first logits
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++) {
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) z[t][r] = fmaf(z[t][r], a.to_log2, -reference[t]);
                }
                if (m0 + 16 > end) {
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++)
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++)
                            if (m0 + 4 * q + r >= end) z[t][r] = -infinity;
                }
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++) {
                    top[t] = fmaxf(fmaxf(z[t][0], z[t][1]), fmaxf(z[t][2], z[t][3]));
                    above |= top[t] > far_above || (!begun[t] && top[t] > -infinity);
                }
                // a lane's first logits, or ones far above its reference: they become the reference
                if (__any(above)) {
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++) {
                        const bool begins = !begun[t] && top[t] > -infinity, moves = begins || top[t] > far_above;
                        const float to = reference[t] + top[t];
                        if (begun[t] && moves) sum[t] *= __builtin_amdgcn_exp2f(reference[t] - to);
                        if (moves) z[t] -= to - reference[t];
                        reference[t] = moves ? to : reference[t];
                        begun[t] |= begins;
                    }
                }
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++)
                    sum[t] += (__builtin_amdgcn_exp2f(z[t][0]) + __builtin_amdgcn_exp2f(z[t][1])) + (__builtin_amdgcn_exp2f(z[t][2]) + __builtin_amdgcn_exp2f(z[t][3]));
            } else {
                floatx4 first{}, factor{};
                uintx4 hits{};
                bool hit = false;
                if constexpr (own_table) {
                    first = *reinterpret_cast<const floatx4*>(row_first + mt * 16 + 4 * q);
                    factor = *reinterpret_cast<const floatx4*>(row_factor + mt * 16 + 4 * q);
                    hits = *reinterpret_cast<const uintx4*>(row_target + mt * 16 + 4 * q);
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) hit |= hits[r] - own_first < TILES * 16u;
                } else {
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++) hit |= target[t] - m0 < 16u;
                }
                bf16x4 y[DT][PARTS];
#pragma unroll
                for (uint32_t d = 0; d < DT; d++)
#pragma unroll
                    for (uint32_t part = 0; part < PARTS; part++) {
                        using Four = __attribute__((address_space(3))) shortx4;
                        y[d][part] = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Four*)(lds + part * part_bytes + column_at[d] + mt * 256)));
                    }
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++)
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) {
                        z[t][r] = __builtin_amdgcn_exp2f(fmaf(z[t][r], a.to_log2, -(own_table ? first[r] : own_lse[t])));
                        if constexpr (own_table) z[t][r] *= factor[r];
                    }
                if (!own_table && m0 + 16 > end) {  // (past the table: a zero less the log sum may be an exponential without bounds)
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++)
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++)
                            if (m0 + 4 * q + r >= end) z[t][r] = 0.0f;
                }
                if (__any(hit)) {
                    floatx4 weight{};
                    if constexpr (own_table) weight = *reinterpret_cast<const floatx4*>(row_weight + mt * 16 + 4 * q);
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++)
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++) {
                            const bool is_target = own_table ? hits[r] == own_first + t * 16 + e : target[t] == m0 + 4 * q + r;
                            if (is_target) z[t][r] -= own_table ? weight[r] : own_one[t];
                        }
                }
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++) {
                    constexpr uint32_t g_parts = PARTS == 3 ? 3 : 2;
                    bf16x4 g[g_parts];
                    const float x[4] = {z[t][0], z[t][1], z[t][2], z[t][3]};
                    entropy_split<g_parts>(g, x);
#pragma unroll
                    for (uint32_t d = 0; d < DT; d++) {
                        out[t][d] = multiply(pair(y[d][0], y[d][0]), pair(g[0], g[1]), out[t][d]);
                        if constexpr (PARTS >= 2) out[t][d] = multiply(pair(y[d][1], y[d][1]), pair(g[0], g[1]), out[t][d]);
                        if constexpr (PARTS == 3) out[t][d] = multiply(pair(y[d][0], y[d][2]), pair(g[2], g[0]), out[t][d]);
                    }
                }
            }
        }
    }

    const uint64_t split_at = blockIdx.y * stream_waves + stream_wave;
#pragma unroll
    for (uint32_t t = 0; t < TILES; t++) {
        const uint32_t o = own_first + t * 16 + e;
        if constexpr (!gradient) {
            float top = begun[t] ? reference[t] : -infinity, total = sum[t];
#pragma unroll
            for (uint32_t x = 16; x < 64; x <<= 1) {
                const float other = __shfl_xor(top, x), other_total = __shfl_xor(total, x);
                const float higher = fmaxf(top, other), base = higher == -infinity ? 0.0f : higher;
                total = total * __builtin_amdgcn_exp2f(top - base) + other_total * __builtin_amdgcn_exp2f(other - base);
                top = higher;
            }
            if (q == 0 && o < own_end) a.partial[split_at * a.padded + o] = make_float2(top, total);
            if (split_at == 0 && q == 0 && o < own_end) {
                float dot = 0.0f;
                for (uint32_t k = 0; k < a.columns; k++)
                    dot = fmaf(static_cast<float>(own[o * own_stride + k]), static_cast<float>(stream[static_cast<uint64_t>(target[t]) * stream_stride + k]), dot);
                a.target_logit[o] = dot * a.to_log2;
            }
        } else if (o < own_end) {
#pragma unroll
            for (uint32_t d = 0; d < DT; d++) {
                const uint32_t column = d * 16 + 4 * q;
                if (column < a.slab_stride)
                    *reinterpret_cast<floatx4*>(a.slab + (split_at * a.slab_rows + o) * a.slab_stride + column) = own_table ? out[t][d] : out[t][d] * own_factor[t];
            }
        }
    }
}

// tiles of owned rows a wave: as many as its registers hold
constexpr uint32_t tiles_of(uint32_t blocks, uint32_t parts) { return blocks <= 2 ? 4 : blocks <= 6 || parts < 3 ? 2 : 1; }

template <typename T, EntropyProduct P, int KB>
void launch(const EntropyNarrowArgs& a, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((entropy_narrow_kernel<T, P, KB, tiles_of(KB, parts_of<T>)>), grid, dim3(block), 0, s, a);
}

// column blocks that kernels are made for
uint32_t blocks_of(uint32_t columns) {
    const uint32_t blocks = (columns + 7) / 8;
    return blocks <= 2 ? blocks : blocks <= 4 ? 4 : blocks <= 6 ? 6 : 8;
}

template <typename T, EntropyProduct P>
void with_columns(const EntropyNarrowArgs& a, dim3 grid, hipStream_t s) {
    switch (blocks_of(a.columns)) {
        case 1: launch<T, P, 1>(a, grid, s); break;
        case 2: launch<T, P, 2>(a, grid, s); break;
        case 4: launch<T, P, 4>(a, grid, s); break;
        case 6: launch<T, P, 6>(a, grid, s); break;
        default: launch<T, P, 8>(a, grid, s); break;
    }
}

template <typename T>
void with_product(EntropyProduct product, const EntropyNarrowArgs& a, dim3 grid, hipStream_t s) {
    if (product == entropy_logits) with_columns<T, entropy_logits>(a, grid, s);
    else if (product == entropy_features_gradient) with_columns<T, entropy_features_gradient>(a, grid, s);
    else with_columns<T, entropy_table_gradient>(a, grid, s);
}

}  // namespace

EntropyNarrowPlan entropy_narrow_plan(uint32_t own, uint32_t stream, uint32_t columns, int type) {
    const uint32_t parts = type == type_float ? parts_of<float> : type == type_bfloat16 ? parts_of<__bf16> : parts_of<_Float16>;
    const uint32_t wave_rows = tiles_of(blocks_of(columns), parts) * 16;
    EntropyNarrowPlan p{};
    p.own_waves = own > 2 * wave_rows ? 4 : own > wave_rows ? 2 : 1;
    p.blocks = std::max(div_up(own, p.own_waves * wave_rows), 1u);
    // Blocks for four to a CU, unless one would meet fewer than four chunks; and none that meets many more than 64 (sums of 4,096 rows; one of 15,000 in a row
    // cost as much precision as all else: table gradient of 1M x 4,096 x 8 1.8e-6 off in 64 parts), where the partial sums take 128 MB at most.
    const uint64_t chunks = std::max(div_up(stream, chunk), 1u), waves_beside = waves / p.own_waves;
    const uint64_t wanted = std::max<uint64_t>(1024u / p.blocks, (chunks + 63) / 64);
    const uint64_t room = (128ull << 20) / (static_cast<uint64_t>(own) * std::max(columns, 4u) * sizeof(float) * waves_beside + 1);
    p.stream_blocks = static_cast<uint32_t>(std::max<uint64_t>(1, std::min({wanted, (chunks + 3) / 4, std::max<uint64_t>(room, 1024u / p.blocks), uint64_t{1024}})));
    p.splits = p.stream_blocks * (waves / p.own_waves);
    return p;
}

void launch_entropy_narrow(EntropyProduct product, int type, const EntropyNarrowArgs& args, const EntropyNarrowPlan& p, hipStream_t s) {
    EntropyNarrowArgs a = args;
    a.own_waves = p.own_waves;
    const dim3 grid(p.blocks, p.stream_blocks);
    if (type == type_float) with_product<float>(product, a, grid, s);
    else if (type == type_bfloat16) with_product<__bf16>(product, a, grid, s);
    else with_product<_Float16>(product, a, grid, s);
}

}  // namespace efgs
