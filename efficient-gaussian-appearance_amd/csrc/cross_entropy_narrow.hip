// The cross entropy for rows of few columns (codes): the logits of a tile of both sides never leave the registers.
//
// A wave owns up to 64 rows of one side, 16 to a tile, and meets the rows of the other side 16 at a time, from LDS:
//   logits      S(m, o) = sum_k stream(m, k) own(o, k)        v_mfma_f32_16x16x4_f32, a lane has four m at one o
//   gradient    out(d, o) += sum_m stream(m, d) g(m, o)       g's registers as they lie are this product's operand: register r of lane (o, q) is row 4 q + r
// The forward and the rows' gradient own packed rows and meet the table; the table's gradient owns table rows and meets the packed rows. The owned side
// comes times scale log2 e, so that a product goes into the exponential less its row's log sum (in the forward, less the lane's reference). Sums that several blocks or waves share are left as partial ones, joined in their order.
#include <algorithm>

#include "cross_entropy.h"

namespace efgs {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

template <typename T, int W> using Part = T __attribute__((ext_vector_type(W), aligned(sizeof(T))));

constexpr uint32_t block = 256, waves = 4, chunk = 64, chunk_tiles = chunk / 16;
constexpr float infinity = __builtin_inff();
constexpr float far_above = 64.0f;   // how far (log 2) a logit may lie above the lane's reference: what sums of 2^64 and below leave room for

__device__ __forceinline__ uint32_t scalar(uint32_t x) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x))); }

// four consecutive values, those from `valid` on zero
template <typename T>
__device__ __forceinline__ floatx4 load4(const T* p, int32_t valid) {
    floatx4 x{};
    if (valid >= 4) {
        const Part<T, 4> v = *reinterpret_cast<const Part<T, 4>*>(p);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = static_cast<float>(v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = k < valid ? static_cast<float>(p[k]) : 0.0f;
    }
    return x;
}

// KS: steps of four columns; DT: tiles of 16 columns; TILES: of 16 owned rows a wave
template <typename T, EntropyProduct P, int KS, int DT, int TILES>
__global__ __launch_bounds__(block) void entropy_narrow_kernel(EntropyNarrowArgs a) {
    constexpr bool gradient = P != entropy_logits, own_table = P == entropy_table_gradient;
    constexpr uint32_t pitch = DT * 16 + 4, quads = KS <= 4 ? 1 : KS / 4;  // (row 4 q + r: four q in four parts of the banks)
    __shared__ float logit_tiles[chunk * KS * 4];                                          // tile, step, lane
    __shared__ __attribute__((aligned(16))) float rows[gradient ? chunk * pitch : 4];       // row-major, of the table's gradient times their weights
    __shared__ __attribute__((aligned(16))) float row_lse[2][own_table ? chunk : 4];
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

    float fo[TILES][KS];
    float2 lse[TILES];
    uint32_t target[TILES];
    floatx4 out[TILES][DT];
    float reference[TILES], sum[TILES];
    bool begun[TILES];
#pragma unroll
    for (uint32_t t = 0; t < TILES; t++) {
        const uint32_t o = own_first + t * 16 + e;
        const bool inside = o < own_end;
#pragma unroll
        for (uint32_t s = 0; s < KS; s++)
            fo[t][s] = inside && 4 * s + q < a.columns ? static_cast<float>(own[o * own_stride + 4 * s + q]) * a.to_log2 : 0.0f;
        lse[t] = P == entropy_features_gradient && inside ? a.lse[o] : make_float2(0.0f, 0.0f);
        target[t] = !own_table && inside ? a.target[o] : entropy_none;
        reference[t] = 0.0f;
        begun[t] = false;
        sum[t] = 0.0f;
#pragma unroll
        for (uint32_t d = 0; d < DT; d++) out[t][d] = floatx4{};
    }

    // a chunk of the streamed rows on its way to the registers: row threadIdx.x / 4, every fourth quad of its columns
    const uint32_t row = threadIdx.x / 4, quad = threadIdx.x % 4;
    floatx4 next[quads];
    float2 next_lse{};
    float next_weight = 0.0f;
    uint32_t next_target = entropy_none;
    const auto fetch = [&](uint32_t from) {
        const uint32_t m = from + row;
#pragma unroll
        for (uint32_t j = 0; j < quads; j++) {
            const uint32_t column = (quad + 4 * j) * 4;
            next[j] = load4<T>(stream + static_cast<uint64_t>(m) * stream_stride + column, m < stream_end ? static_cast<int32_t>(a.columns) - static_cast<int32_t>(column) : 0);
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
        for (uint32_t j = 0; j < quads; j++) {
            const uint32_t s = quad + 4 * j;
            if (s < KS) {
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) logit_tiles[((row / 16) * KS + s) * 64 + k * 16 + row % 16] = next[j][k];
                if constexpr (gradient) *reinterpret_cast<floatx4*>(rows + row * pitch + s * 4) = own_table ? next[j] * next_weight : next[j];
            }
        }
        if constexpr (own_table) {
            if (quad == 0) {
                row_lse[0][row] = next_lse.x;
                row_lse[1][row] = next_lse.y;
                row_target[row] = next_target;
            }
        }
        __syncthreads();
        if (from + chunk < end) fetch(from + chunk);
        if constexpr (!gradient) {
            for (uint32_t mt = stream_wave; mt < chunk_tiles; mt += stream_waves) {
                if (from + mt * 16 >= end) break;
                float fs[KS];
#pragma unroll
                for (uint32_t s = 0; s < KS; s++) fs[s] = logit_tiles[(mt * KS + s) * 64 + lane];
                floatx4 z[TILES];
                bool above = false;
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++) {
                    z[t] = floatx4{};
#pragma unroll
                    for (uint32_t s = 0; s < KS; s++) z[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(fs[s], fo[t][s], z[t], 0, 0, 0);
                }
                if (from + mt * 16 + 16 > end) {
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++)
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++)
                            if (from + mt * 16 + 4 * q + r >= end) z[t][r] = -infinity;
                }
                float top[TILES];  // above the reference, or the first logits
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++) {
                    z[t] -= reference[t];
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
            }
        } else {
            for (uint32_t mt = stream_wave; mt < chunk_tiles; mt += stream_waves) {
                const uint32_t m0 = from + mt * 16;
                if (m0 >= end) break;
                float fs[KS], fr[4][DT];
#pragma unroll
                for (uint32_t s = 0; s < KS; s++) fs[s] = logit_tiles[(mt * KS + s) * 64 + lane];
#pragma unroll
                for (uint32_t r = 0; r < 4; r++)
#pragma unroll
                    for (uint32_t d = 0; d < DT; d++) fr[r][d] = rows[(mt * 16 + 4 * q + r) * pitch + d * 16 + e];
                floatx4 first{}, second{};
                uintx4 hits{};
                bool hit = false;
                if constexpr (own_table) {
                    first = *reinterpret_cast<const floatx4*>(row_lse[0] + mt * 16 + 4 * q);
                    second = *reinterpret_cast<const floatx4*>(row_lse[1] + mt * 16 + 4 * q);
                    hits = *reinterpret_cast<const uintx4*>(row_target + mt * 16 + 4 * q);
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) hit |= hits[r] - own_first < TILES * 16u;
                } else {
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++) hit |= target[t] - m0 < 16u;
                }
                floatx4 p[TILES];
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++) {
                    p[t] = floatx4{};
#pragma unroll
                    for (uint32_t s = 0; s < KS; s++) p[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(fs[s], fo[t][s], p[t], 0, 0, 0);
                }
#pragma unroll
                for (uint32_t t = 0; t < TILES; t++)
#pragma unroll
                    for (uint32_t r = 0; r < 4; r++) p[t][r] = __builtin_amdgcn_exp2f((p[t][r] - (own_table ? first[r] : lse[t].x)) - (own_table ? second[r] : lse[t].y));
                if (!own_table && m0 + 16 > end) {  // (past the table: a zero less the log sum may be an exponential without bounds)
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++)
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++)
                            if (m0 + 4 * q + r >= end) p[t][r] = 0.0f;
                }
                if (__any(hit)) {
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++)
#pragma unroll
                        for (uint32_t r = 0; r < 4; r++) {
                            const bool is_target = own_table ? hits[r] == own_first + t * 16 + e : target[t] == m0 + 4 * q + r;
                            if (is_target) p[t][r] -= 1.0f;
                        }
                }
#pragma unroll
                for (uint32_t r = 0; r < 4; r++)
#pragma unroll
                    for (uint32_t t = 0; t < TILES; t++)
#pragma unroll
                        for (uint32_t d = 0; d < DT; d++) out[t][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(fr[r][d], p[t][r], out[t][d], 0, 0, 0);
            }
        }
    }

    const uint64_t split = blockIdx.y * stream_waves + stream_wave;
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
            if (q == 0 && o < own_end) a.partial[split * a.padded + o] = make_float2(top, total);
            if (split == 0 && q == 0 && o < own_end) {
                float z = 0.0f;
                for (uint32_t k = 0; k < a.columns; k++)
                    z = fmaf(static_cast<float>(own[o * own_stride + k]) * a.to_log2, static_cast<float>(stream[static_cast<uint64_t>(target[t]) * stream_stride + k]), z);
                a.target_logit[o] = z;
            }
        } else if (o < own_end) {
            // (q's sums of the wave are whole: the product's k is over q)
#pragma unroll
            for (uint32_t d = 0; d < DT; d++) {
                const uint32_t column = d * 16 + 4 * q;
                if (column < a.slab_stride) *reinterpret_cast<floatx4*>(a.slab + (split * a.slab_rows + o) * a.slab_stride + column) = out[t][d];
            }
        }
    }
}

template <typename T, EntropyProduct P, int KS, int TILES>
void launch(const EntropyNarrowArgs& a, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((entropy_narrow_kernel<T, P, KS, (KS + 3) / 4, TILES>), grid, dim3(block), 0, s, a);
}

template <typename T, EntropyProduct P>
void with_columns(const EntropyNarrowArgs& a, dim3 grid, hipStream_t s) {
    const uint32_t steps = (a.columns + 3) / 4;
    if (steps <= 1) launch<T, P, 1, 4>(a, grid, s);
    else if (steps <= 2) launch<T, P, 2, 4>(a, grid, s);
    else if (steps <= 4) launch<T, P, 4, 4>(a, grid, s);
    else if (steps <= 8) launch<T, P, 8, 4>(a, grid, s);
    else if (steps <= 12) launch<T, P, 12, 4>(a, grid, s);
    else if (steps <= 16) launch<T, P, 16, 4>(a, grid, s);
    else if (steps <= 24) launch<T, P, 24, 2>(a, grid, s);
    else launch<T, P, 32, 2>(a, grid, s);
}

template <typename T>
void with_product(EntropyProduct product, const EntropyNarrowArgs& a, dim3 grid, hipStream_t s) {
    if (product == entropy_logits) with_columns<T, entropy_logits>(a, grid, s);
    else if (product == entropy_features_gradient) with_columns<T, entropy_features_gradient>(a, grid, s);
    else with_columns<T, entropy_table_gradient>(a, grid, s);
}

}  // namespace

EntropyNarrowPlan entropy_narrow_plan(uint32_t own, uint32_t stream, uint32_t columns) {
    const uint32_t wave_rows = columns <= 64 ? 64 : 32;
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
