// Softmax cross entropy of rows x_n against every row w_v of a table, without the logits in memory, and its gradients:
//
//   z_nv = scale x_n . w_v,  loss_n = log sum_v exp z_nv - z_n,target(n)
//   g_nv = upstream_n (p_nv - [v = target(n)]),  dx_n = scale sum_v g_nv w_v,  dw_v = scale sum_n g_nv x_n
//
// A target outside the table leaves its row out. The rows that count are packed first (in their order, columns padded with
// zeros), so that rows left out cost nothing behind that and nothing that stands in them reaches a sum. The forward is one
// matrix product whose tiles leave, for each row, the maximum and the sum of exponentials over the tile's part of the table; a
// second kernel joins them. The backward computes the logits again by pieces of the table, writes g of a piece, and multiplies
// it by the piece and, transposed, by the rows: four products where three would do if g could be kept (N x V of it), and no more memory than a piece.
// Statistics and sums are in 32 bits (logits in units of log 2), the sum over rows in 64. g is held in the inputs' type, as the matrix unit takes it (floats: three
// bfloat16 parts): its rounding, bfloat16 2^-8 of each at most, is as large as the gradients' own one only where one entry outweighs the others, which a row's
// target does; what that one loses is added (cross_entropy_wide.hip).
//
// This file: the packing, the joins and the launches, most of them at the latency of a launch, 4 to 9 us each. The products: cross_entropy_narrow.hip up to 64
// columns, where its kernels are the faster ones (32,768 x 4,096 x 64: float32 0.66 ms and 1.07 by the wide one, bfloat16 0.24 and 0.34; float16 0.41 and 0.35, for
// no piece in memory); cross_entropy_wide.hip above, as a wave's rows would not fit the narrow ones' registers; up to 64 rows without a gradient
// cross_entropy_few.hip, which no packing precedes (37 x 30,011 x 1,000 float16 40 us by the wide one, 24 so).
#include <algorithm>
#include <type_traits>

#include "cross_entropy.h"

namespace efgs {

namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr float log2_e = 1.4426950408889634f, ln_2 = 0.6931471805599453f, infinity = __builtin_inff();
constexpr uint32_t none = entropy_none, row_tile = entropy_row_tile, column_tile = entropy_column_tile;
constexpr uint32_t rank_block = 1024;
constexpr uint32_t count_alone = 16384;   // largest list that every block counts by itself

template <typename T, int W> using Part = T __attribute__((ext_vector_type(W), aligned(sizeof(T))));

uint64_t round_up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }

// ---- the rows that count ---------------------------------------------------------------------------------------------

struct Packing {
    const void* targets;
    uint32_t n, padded, rows, target_bytes;
    uint32_t* chunk_counts;  // null: short lists
    uint32_t* count;         // rows that count
    uint32_t* row_of;        // packed row -> row
    uint32_t* packed_of;     // row -> packed row, or none
    uint32_t* target;        // of a packed row; none past them
};

__device__ __forceinline__ uint32_t target_at(const Packing& a, uint32_t i) {
    const int64_t t = a.target_bytes == 8 ? static_cast<const int64_t*>(a.targets)[i] : static_cast<const int32_t*>(a.targets)[i];
    return static_cast<uint64_t>(t) < a.rows ? static_cast<uint32_t>(t) : none;
}

__device__ __forceinline__ uint32_t block_total(uint32_t v, uint32_t* lds) {
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    uint32_t sum = 0;
    for (uint32_t w = 0; w < rank_block / 64; w++) sum += lds[w];
    return sum;
}

__global__ __launch_bounds__(rank_block) void entropy_count_kernel(Packing a) {
    __shared__ uint32_t lds[rank_block / 64];
    const uint32_t i = blockIdx.x * rank_block + threadIdx.x;
    const uint32_t total = block_total(i < a.n && target_at(a, i) != none, lds);
    if (threadIdx.x == 0) a.chunk_counts[blockIdx.x] = total;
}

// a block a chunk of rank_block rows
__global__ __launch_bounds__(rank_block) void entropy_rank_kernel(Packing a) {
    __shared__ uint32_t lds[rank_block / 64], waves[rank_block / 64];
    uint32_t before = 0, all = 0;
    if (a.chunk_counts) {
        for (uint32_t c = threadIdx.x; c < gridDim.x; c += rank_block) {
            const uint32_t k = a.chunk_counts[c];
            all += k;
            before += c < blockIdx.x ? k : 0u;
        }
    } else {
        for (uint32_t i = threadIdx.x; i < a.n; i += rank_block) {
            const bool counts = target_at(a, i) != none;
            all += counts;
            before += counts && i < blockIdx.x * rank_block;
        }
    }
    before = block_total(before, lds);
    all = block_total(all, lds);
    const uint32_t i = blockIdx.x * rank_block + threadIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t target = i < a.n ? target_at(a, i) : none;
    const uint64_t ballot = __ballot(target != none);
    if (lane == 0) waves[wave] = static_cast<uint32_t>(__popcll(ballot));
    __syncthreads();
    uint32_t at = before + static_cast<uint32_t>(__popcll(ballot & ((1ull << lane) - 1ull)));
    for (uint32_t w = 0; w < wave; w++) at += waves[w];
    if (i < a.n) a.packed_of[i] = target == none ? none : at;
    if (target != none) {
        a.row_of[at] = i;
        a.target[at] = target;
    }
    if (i >= all && i < a.padded) {
        a.row_of[i] = none;
        a.target[i] = none;
    }
    if (i == 0) *a.count = all;
}

struct Copying {
    const void* from;
    uint64_t stride;
    uint32_t rows, columns, padded_columns;
    const uint32_t* count;   // packed rows, or null: all
    const uint32_t* row_of;
    void* to;
};

// Rows with their columns padded by zeros, sixteen bytes a thread. Of packed rows, those past the ones that count are zeros, up to a whole tile.
template <typename T>
__global__ __launch_bounds__(256) void entropy_copy_kernel(Copying a) {
    constexpr uint32_t W = 16 / sizeof(T);
    const uint32_t parts = a.padded_columns / W, end = a.count ? (*a.count + row_tile - 1) / row_tile * row_tile : a.rows;
    const uint64_t items = static_cast<uint64_t>(end) * parts, step = static_cast<uint64_t>(gridDim.x) * 256u;
    for (uint64_t t = blockIdx.x * 256ull + threadIdx.x; t < items; t += step) {
        const uint32_t m = static_cast<uint32_t>(t / parts), column = static_cast<uint32_t>(t - static_cast<uint64_t>(m) * parts) * W;
        const uint32_t row = a.row_of ? a.row_of[m] : m;
        Part<T, W> v{};
        if (row != none && column < a.columns) {
            const T* const p = static_cast<const T*>(a.from) + row * a.stride + column;
            if (column + W <= a.columns) v = *reinterpret_cast<const Part<T, W>*>(p);
            else
#pragma unroll
                for (uint32_t k = 0; k < W; k++)
                    if (column + k < a.columns) v[k] = p[k];
        }
        *reinterpret_cast<Part<T, W>*>(static_cast<T*>(a.to) + t * W) = v;
    }
}

// Rows of floats as three bfloat16 parts, one after the other, each padded by zeros: eight columns a thread.
__global__ __launch_bounds__(256) void entropy_split_kernel(Copying a) {
    typedef __bf16 Eight __attribute__((ext_vector_type(8)));
    const uint32_t pieces = a.padded_columns / 8, end = a.count ? (*a.count + row_tile - 1) / row_tile * row_tile : a.rows;
    const uint64_t items = static_cast<uint64_t>(end) * pieces, step = static_cast<uint64_t>(gridDim.x) * 256u;
    for (uint64_t t = blockIdx.x * 256ull + threadIdx.x; t < items; t += step) {
        const uint32_t m = static_cast<uint32_t>(t / pieces), column = static_cast<uint32_t>(t - static_cast<uint64_t>(m) * pieces) * 8;
        const uint32_t row = a.row_of ? a.row_of[m] : m;
        float x[8];
        entropy_load8(x, static_cast<const float*>(a.from) + row * a.stride + column,
                      row != none && column < a.columns ? static_cast<int32_t>(a.columns - column) : 0);
        Eight parts[3];
        entropy_split<3>(parts, x);
#pragma unroll
        for (uint32_t k = 0; k < 3; k++)
            *reinterpret_cast<Eight*>(static_cast<__bf16*>(a.to) + (static_cast<uint64_t>(m) * 3 + k) * a.padded_columns + column) = parts[k];
    }
}

// ---- joins -----------------------------------------------------------------------------------------------------------

struct JoinArgs {
    const float2* partial;
    uint32_t tiles;
    uint32_t first_row, rows;  // of packed rows: a launch's
    uint32_t n;
    const uint32_t* count;
    const uint32_t* row_of;
    const uint32_t* packed_of;
    const float* target_logit;
    float2* lse;
    float* losses;         // of each row, or null
    double* sums;          // of each block's rows
};

constexpr uint32_t join_rows = 64;
constexpr uint32_t join_parts = 16, join_alone = 4;  // parts of the tiles; up to so many tiles: one, four times the rows

// 64 packed rows a wave, the tiles of the table in PARTS parts
template <uint32_t PARTS>
__global__ __launch_bounds__(PARTS > 1 ? join_rows * PARTS : 256) void entropy_join_kernel(JoinArgs a) {
    __shared__ float2 parts[PARTS][join_rows];
    const uint32_t lane = threadIdx.x & (join_rows - 1u), wave = threadIdx.x / join_rows, part = PARTS > 1 ? wave : 0;
    const uint32_t at = PARTS > 1 ? blockIdx.x * join_rows + lane : blockIdx.x * 256 + threadIdx.x, row = a.first_row + at;
    const uint32_t count = *a.count;
    const bool counts = row < count;
    float top = -infinity, sum = 0.0f;
    if (counts)
        for (uint32_t t = part; t < a.tiles; t += PARTS) {
            const float2 x = a.partial[static_cast<uint64_t>(t) * a.rows + at];
            const float higher = fmaxf(top, x.x), from = higher == -infinity ? 0.0f : higher;
            sum = sum * __builtin_amdgcn_exp2f(top - from) + x.y * __builtin_amdgcn_exp2f(x.x - from);
            top = higher;
        }
    if constexpr (PARTS > 1) {
        parts[part][lane] = make_float2(top, sum);
        __syncthreads();
        if (part != 0) return;
    }
    for (uint32_t k = 1; k < PARTS; k++) {
        const float2 x = parts[k][lane];
        const float higher = fmaxf(top, x.x), from = higher == -infinity ? 0.0f : higher;
        sum = sum * __builtin_amdgcn_exp2f(top - from) + x.y * __builtin_amdgcn_exp2f(x.x - from);
        top = higher;
    }
    // the sum's power of two joins the reference, with what that sum rounds off
    int exponent = 0;
    const float fraction = sum > 0.0f && sum < infinity ? frexpf(sum, &exponent) : sum;
    const float power = static_cast<float>(exponent), first = top + power, second = log2f(fraction) + (exponent != 0 ? top - (first - power) : 0.0f);
    const float loss = counts ? ((first - a.target_logit[row]) + second) * ln_2 : 0.0f;
    if (counts) a.lse[row] = make_float2(first, second);
    if (a.losses) {
        if (counts) a.losses[a.row_of[row]] = loss;
        if (row < a.n && a.packed_of[row] == none) a.losses[row] = 0.0f;
        return;
    }
    double total = loss;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o);
    if (lane == 0) a.sums[row / join_rows] = total;
}

constexpr uint32_t total_block = 1024;

__global__ __launch_bounds__(total_block) void entropy_total_kernel(const double* sums, uint32_t waves, const uint32_t* count, bool mean, float* loss) {
    __shared__ double lds[total_block / 64];
    double total = 0.0;
    for (uint32_t b = threadIdx.x; b < waves; b += total_block) total += sums[b];
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o);
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = total;
    __syncthreads();
    if (threadIdx.x == 0) {
        total = 0.0;
        for (uint32_t w = 0; w < total_block / 64; w++) total += lds[w];
        *loss = static_cast<float>(mean ? total / max(*count, 1u) : total);
    }
}

// ---- backward's ends ---------------------------------------------------------------------------------------------------

struct WeightArgs {
    const float* upstream;   // one, or one for each row
    const uint32_t* count;
    const uint32_t* row_of;
    uint32_t padded;
    bool each, mean;
    float scale;
    float held;              // what the logits' gradients are held times
    float* weight;           // of packed rows, times `held`
    float* factor;           // of the sums
};

__global__ __launch_bounds__(256) void entropy_weights_kernel(WeightArgs a) {
    const uint32_t m = blockIdx.x * 256 + threadIdx.x, count = *a.count;
    if (m < a.padded) a.weight[m] = m >= count ? 0.0f : (a.each ? a.upstream[a.row_of[m]] : 1.0f) * a.held;
    if (m == 0) *a.factor = (a.each ? a.scale : a.scale * *a.upstream / (a.mean ? static_cast<float>(max(count, 1u)) : 1.0f)) / a.held;
}

// float16, a weight for each row: the weights over the power of two at or above the largest finite one, so that a product of weight and
// probability keeps to the type's range (a row of an infinite one or NaN alone, as the plain product would have it): held times 2^15, each to 2^-39 of the
// largest weight, so that the entries of a row of a far smaller one have fewer bits than float16's eleven. One block.
__global__ __launch_bounds__(1024) void entropy_half_weights_kernel(WeightArgs a) {
    __shared__ float lds[16];
    const uint32_t count = *a.count;
    float top = 0.0f;
    for (uint32_t m = threadIdx.x; m < count; m += 1024) {
        const float weight = fabsf(a.upstream[a.row_of[m]]);
        if (weight < infinity) top = fmaxf(top, weight);
    }
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
    for (uint32_t w = 0; w < 16; w++) top = fmaxf(top, lds[w]);
    int exponent = 0;
    if (top > 0.0f) frexpf(top, &exponent);
    for (uint32_t m = threadIdx.x; m < a.padded; m += 1024)
        a.weight[m] = m < count ? ldexpf(a.upstream[a.row_of[m]], -exponent) * a.held : 0.0f;
    if (threadIdx.x == 0) *a.factor = ldexpf(a.scale / a.held, exponent);
}

struct Gathering {
    const float* slab;           // splits x slab_rows x slab_stride
    uint64_t slab_rows;
    uint32_t slab_stride, splits;
    const uint32_t* packed_of;   // or null: the rows themselves
    const float* weight;         // of packed rows, or null
    const float* residual;       // of packed rows, times their target's table row, or null
    const uint32_t* target;
    const void* table;
    uint64_t table_stride;
    uint32_t rows, columns;
    const float* factor;
};

// four columns of a packed row's own target's table row
template <typename T>
__device__ __forceinline__ floatx4 target_columns(const Gathering& a, uint32_t m, uint32_t column) {
    const T* const p = static_cast<const T*>(a.table) + a.target[m] * a.table_stride + column;
    floatx4 x{};
    if (column + 4 <= a.columns) {
        const Part<T, 4> v = *reinterpret_cast<const Part<T, 4>*>(p);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) x[k] = static_cast<float>(v[k]);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) x[k] = column + k < a.columns ? static_cast<float>(p[k]) : 0.0f;
    }
    return x;
}

// Sums of the splits, in their order, scaled; rows without a packed one are zeros. Four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void entropy_gather_kernel(Gathering a, T* out) {
    const uint32_t parts = (a.columns + 3) / 4, lanes = min(parts, 256u), rows = 256u / lanes, r = threadIdx.x / lanes, lane = threadIdx.x - r * lanes;
    if (r >= rows) return;
    const float factor = *a.factor;
    for (uint64_t row = static_cast<uint64_t>(blockIdx.x) * rows + r; row < a.rows; row += static_cast<uint64_t>(gridDim.x) * rows) {
        const uint32_t m = a.packed_of ? a.packed_of[row] : static_cast<uint32_t>(row);
        const float f = a.weight && m != none ? factor * a.weight[m] : factor;
        for (uint32_t part = lane; part < parts; part += lanes) {
            floatx4 sum{};
            if (m != none)
                for (uint32_t s = 0; s < a.splits; s++)
                    sum += *reinterpret_cast<const floatx4*>(a.slab + (s * a.slab_rows + m) * a.slab_stride + part * 4);
            if (a.residual && m != none) sum += a.residual[m] * target_columns<T>(a, m, part * 4);
            Part<T, 4> y;
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) y[k] = static_cast<T>(m == none ? 0.0f : sum[k] * f);
            T* const to = out + row * a.columns + part * 4;
            if (part * 4 + 4 <= a.columns) *reinterpret_cast<Part<T, 4>*>(to) = y;
            else
#pragma unroll
                for (uint32_t k = 0; k < 4; k++)
                    if (part * 4 + k < a.columns) to[k] = y[k];
        }
    }
}

// The same where there are many splits of few rows: sixteen items of four columns a block, their splits in sixteen parts.
template <typename T>
__global__ __launch_bounds__(256) void entropy_gather_splits_kernel(Gathering a, T* out) {
    __shared__ floatx4 lds[16][16];
    const uint32_t parts = (a.columns + 3) / 4, item = threadIdx.x & 15u, part = threadIdx.x >> 4;
    const uint64_t items = static_cast<uint64_t>(a.rows) * parts, t = min(blockIdx.x * 16ull + item, items - 1);
    const uint64_t row = t / parts;
    const uint32_t column = static_cast<uint32_t>(t - row * parts) * 4, m = a.packed_of ? a.packed_of[row] : static_cast<uint32_t>(row);
    floatx4 sum{};
    if (m != none)
        for (uint32_t s = part; s < a.splits; s += 16) sum += *reinterpret_cast<const floatx4*>(a.slab + (s * a.slab_rows + m) * a.slab_stride + column);
    lds[part][item] = sum;
    __syncthreads();
    if (part != 0 || blockIdx.x * 16ull + item >= items) return;
    for (uint32_t k = 1; k < 16; k++) sum += lds[k][item];
    if (a.residual && m != none) sum += a.residual[m] * target_columns<T>(a, m, column);
    const float f = m == none ? 0.0f : a.weight ? *a.factor * a.weight[m] : *a.factor;
#pragma unroll
    for (uint32_t k = 0; k < 4; k++)
        if (column + k < a.columns) out[row * a.columns + column + k] = static_cast<T>(m == none ? 0.0f : sum[k] * f);
}

// ---- sizes and buffers -------------------------------------------------------------------------------------------------

// hands out 256-byte aligned parts of a buffer, or, without one, counts them
class Carver {
  public:
    explicit Carver(void* base) : base_(static_cast<char*>(base)) {}
    template <typename T>
    T* take(uint64_t n) {
        char* const p = base_ ? base_ + used_ : nullptr;
        used_ += round_up(std::max<uint64_t>(n, 1) * sizeof(T), 256);
        return reinterpret_cast<T*>(p);
    }
    size_t used() const { return used_; }

  private:
    char* base_;
    size_t used_ = 0;
};

uint32_t type_bytes(int type) { return type == type_float ? 4 : 2; }

// the ways: few rows without a gradient; few columns; the others
bool few(const EntropyArgs& a) { return a.n > 0 && a.n <= entropy_few_most && a.rows > 0 && a.columns > 0; }
bool narrow(const EntropyArgs& a) { return a.columns > 0 && a.columns <= entropy_narrow_most; }
bool in_parts(const EntropyArgs& a) { return a.type == type_float && !narrow(a); }  // floats as three bfloat16
uint32_t parts_of(const EntropyArgs& a) { return in_parts(a) ? 3 : 1; }
uint32_t held_bytes(const EntropyArgs& a) { return in_parts(a) ? 6 : type_bytes(a.type); }  // of an element of the packed rows, of the table's copy and of a piece
bool table_is_copied(const EntropyArgs& a);

struct Saved {
    uint32_t* count;
    uint32_t* row_of;
    uint32_t* packed_of;
    uint32_t* target;
    float2* lse;
    void* packed;
    uint32_t padded, padded_columns;
    size_t bytes;
    Saved(const EntropyArgs& a, void* base) {
        Carver c(base);
        padded = static_cast<uint32_t>(round_up(std::max(a.n, 1u), row_tile));
        padded_columns = static_cast<uint32_t>(round_up(a.columns, narrow(a) ? 16 / type_bytes(a.type) : column_tile));
        count = c.take<uint32_t>(1);
        row_of = c.take<uint32_t>(padded);
        packed_of = c.take<uint32_t>(padded);
        target = c.take<uint32_t>(padded);
        lse = c.take<float2>(padded);
        packed = c.take<char>(static_cast<uint64_t>(padded) * padded_columns * held_bytes(a));
        bytes = c.used();
    }
};

constexpr uint64_t most_blocks = 1ull << 23;      // of a launch of 256 threads (32 bits of threads)
constexpr uint32_t tile = 128;                    // the smaller tiles' side

// The side of a product's tiles, and how often its k is split: where tiles leave much of the GPU idle, smaller ones and more blocks, at the price of less reuse, or of
// partial results (`results` floats) written and read once more for each split. Measured: a CU takes 1.7 us for 64 of k of a tile of 256, 1.2 for those of
// two of 128 (0.8 for one alone); partial results move at 4 TB/s. Floats: six times the steps, and with more than 2^21 columns small tiles, whose rows' parts
// 32 bits of bytes reach over.
struct ProductPlan {
    uint32_t side, splits;
};

ProductPlan plan_product(const EntropyArgs& a, uint64_t i, uint64_t j, uint64_t k, uint64_t results) {
    ProductPlan best{tile, 1};
    double least = 1e30;
    for (const uint32_t side : {256u, 128u}) {
        if (side == 256 && in_parts(a) && a.columns > 1u << 21) continue;
        const uint64_t tiles = ((i + side - 1) / side) * ((j + side - 1) / side), at_once = side == 256 ? 256 : 512, step = 64;
        for (const uint32_t s : {1u, 2u, 3u, 4u, 6u, 8u, 12u, 16u, 24u, 32u, 48u, 64u}) {
            if (s > 1 && (results == 0 || k / s < 2 * step || tiles * s > most_blocks / 4)) break;
            const uint64_t blocks = tiles * s;
            const double step_us = side == 256 ? 1.7 : blocks <= 256 ? 0.8 : 1.2;
            const double rounds = static_cast<double>((blocks + at_once - 1) / at_once);
            const double steps = static_cast<double>((k + s * step - 1) / (s * step) * (in_parts(a) ? 6 : 1));
            const double us = rounds * (steps + 2.0) * step_us + (s > 1 ? s * static_cast<double>(results) * 8.0 / 4e6 : 0.0);
            if (us < least) {
                least = us;
                best = {side, s};
            }
        }
    }
    return best;
}

constexpr uint64_t partial_bytes = 256ull << 20;  // of the tiles' statistics at once
// A piece's upstream gradients take what the memory-side cache holds, but at least 1,024 table rows if 8 GB are enough for them: with less the products' k is
// short and every piece reads and writes the rows' gradient once more (256 and 1,024 rows: 1M x 4,096 x 72 bfloat16 17.3 and 11.6 ms, 200,000 x 4,096 x 200
// float32 16.9 and 11.8; 100,000 x 20,000 x 136 bfloat16 7.1 either way).
constexpr uint64_t piece_bytes = 256ull << 20, piece_most = 8ull << 30;
constexpr uint32_t piece_least = 1024;

struct ForwardScratch {
    uint32_t* chunk_counts;
    float2* partial;
    float* target_logit;
    double* sums;
    void* copy;        // of the table, or null
    bool copied;
    EntropyNarrowPlan plan;
    uint32_t side, tiles, rows_at_once;
    size_t bytes;
    ForwardScratch(const EntropyArgs& a, const Saved& s, void* base) {
        Carver c(base);
        plan = entropy_narrow_plan(std::max(a.n, 1u), a.rows, a.columns, a.type);
        side = plan_product(a, a.rows, s.padded, a.columns, 0).side;
        tiles = narrow(a) ? (a.rows > 0 ? plan.splits : 0) : div_up(a.rows, side);
        chunk_counts = c.take<uint32_t>(div_up(s.padded, rank_block));
        const uint64_t most = std::min(partial_bytes / sizeof(float2), most_blocks * tile) / std::max(tiles, 1u);
        rows_at_once = narrow(a) ? s.padded : static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>(most / row_tile * row_tile, row_tile), s.padded));
        partial = c.take<float2>(static_cast<uint64_t>(tiles) * rows_at_once);
        target_logit = c.take<float>(s.padded);
        sums = c.take<double>(s.padded / join_rows);
        copy = table_is_copied(a) ? c.take<char>(static_cast<uint64_t>(a.rows) * s.padded_columns * held_bytes(a)) : nullptr;
        copied = table_is_copied(a);
        bytes = c.used();
    }
};

struct NarrowBackwardScratch {
    float* weight;
    float* factor;
    float* slab;             // of one gradient after the other
    EntropyNarrowPlan features, table;
    uint32_t slab_stride;
    size_t bytes;
    NarrowBackwardScratch(const EntropyArgs& a, const Saved& s, void* base) {
        Carver c(base);
        features = entropy_narrow_plan(std::max(a.n, 1u), a.rows, a.columns, a.type);
        table = entropy_narrow_plan(a.rows, std::max(a.n, 1u), a.columns, a.type);
        slab_stride = static_cast<uint32_t>(round_up(a.columns, 4));
        weight = c.take<float>(s.padded);
        factor = c.take<float>(1);
        slab = c.take<float>(std::max(static_cast<uint64_t>(features.splits) * s.padded, static_cast<uint64_t>(table.splits) * a.rows) * slab_stride);
        bytes = c.used();
    }
};

struct BackwardScratch {
    float* weight;
    float* factor;
    float* residual;         // of packed rows
    void* piece;
    float* features_slab;
    float* table_slab;
    void* copy;              // of the table, or null
    bool copied;
    uint32_t piece_rows, pieces;
    ProductPlan upstream, features, table;
    size_t bytes;
    BackwardScratch(const EntropyArgs& a, const Saved& s, void* base) {
        Carver c(base);
        const uint64_t row_bytes = static_cast<uint64_t>(s.padded) * held_bytes(a);   // of a table row's part of a piece
        const uint64_t most = std::max<uint64_t>(std::max<uint64_t>(piece_bytes / row_bytes, std::min<uint64_t>(piece_least, piece_most / row_bytes)) / 256 * 256, 256);
        const uint64_t all = round_up(std::max(a.rows, 1u), 256);
        pieces = div_up(all, std::min(most, all));
        piece_rows = static_cast<uint32_t>(round_up(div_up(all, pieces), 256));
        pieces = div_up(all, piece_rows);
        upstream = plan_product(a, piece_rows, s.padded, a.columns, 0);
        features = plan_product(a, a.columns, s.padded, piece_rows, static_cast<uint64_t>(s.padded) * s.padded_columns);
        table = plan_product(a, a.columns, piece_rows, s.padded, static_cast<uint64_t>(piece_rows) * s.padded_columns);
        weight = c.take<float>(s.padded);
        factor = c.take<float>(1);
        residual = c.take<float>(s.padded);
        piece = c.take<char>(static_cast<uint64_t>(s.padded) * piece_rows * held_bytes(a));
        features_slab = c.take<float>(static_cast<uint64_t>(features.splits) * s.padded * s.padded_columns);
        table_slab = table.splits > 1 ? c.take<float>(static_cast<uint64_t>(table.splits) * piece_rows * s.padded_columns) : nullptr;
        copied = table_is_copied(a);
        copy = copied ? c.take<char>(static_cast<uint64_t>(a.rows) * s.padded_columns * held_bytes(a)) : nullptr;
        bytes = c.used();
    }
};

template <typename F>
void with_type(int type, F&& f) {
    if (type == type_float) f(float{});
    else if (type == type_bfloat16) f(__bf16{});
    else f(static_cast<_Float16>(0.0f));
}

constexpr uint32_t copy_blocks = 1u << 16;

uint32_t copy_grid(uint64_t items) { return static_cast<uint32_t>(std::min<uint64_t>(std::max<uint64_t>((items + 255) / 256, 1), copy_blocks)); }

void launch_copy(const EntropyArgs& a, const Copying& c, uint64_t most_rows, hipStream_t stream) {
    if (c.padded_columns == 0 || most_rows == 0) return;
    if (in_parts(a)) {
        hipLaunchKernelGGL(entropy_split_kernel, dim3(copy_grid(most_rows * c.padded_columns / 8)), dim3(256), 0, stream, c);
        return;
    }
    const uint32_t blocks = copy_grid(most_rows * c.padded_columns * type_bytes(a.type) / 16);
    with_type(a.type, [&](auto t) { hipLaunchKernelGGL(entropy_copy_kernel<decltype(t)>, dim3(blocks), dim3(256), 0, stream, c); });
}

void launch_packing(const EntropyArgs& a, const Saved& s, uint32_t* chunk_counts, hipStream_t stream) {
    Packing p{};
    p.targets = a.targets;
    p.n = a.n;
    p.padded = s.padded;
    p.rows = a.rows;
    p.target_bytes = static_cast<uint32_t>(a.target_bytes);
    p.chunk_counts = a.n > count_alone ? chunk_counts : nullptr;
    p.count = s.count;
    p.row_of = s.row_of;
    p.packed_of = s.packed_of;
    p.target = s.target;
    const dim3 chunks(div_up(s.padded, rank_block));
    if (p.chunk_counts) hipLaunchKernelGGL(entropy_count_kernel, chunks, dim3(rank_block), 0, stream, p);
    hipLaunchKernelGGL(entropy_rank_kernel, chunks, dim3(rank_block), 0, stream, p);
    launch_copy(a, Copying{a.features, a.feature_stride, a.n, a.columns, s.padded_columns, s.count, s.row_of, s.packed}, s.padded, stream);
}

// A table whose rows the wide products cannot read as they lie: another alignment than 16 bytes, columns that 16 bytes do not divide, rows that
// overlap, or so far apart that 32 bits of bytes do not reach over a tile; and one of floats, for their parts. A copy takes its place.
bool table_is_copied(const EntropyArgs& a) {
    if (narrow(a) || a.rows == 0) return false;
    return in_parts(a) || (reinterpret_cast<uintptr_t>(a.table) % 16 != 0 || a.columns % 8 != 0 || a.table_stride % 8 != 0 ||
                                     a.table_stride < a.columns || a.table_stride >= 1ull << 22);
}

// the table, or its copy in `room`
struct Table {
    const void* rows;
    uint64_t stride;
    uint32_t columns;   // (of a part)
};

Table table_of(const EntropyArgs& a, const Saved& s, void* room, hipStream_t stream) {
    if (!room) return {a.table, a.table_stride, a.columns};
    launch_copy(a, Copying{a.table, a.table_stride, a.rows, a.columns, s.padded_columns, nullptr, nullptr, room}, a.rows, stream);
    return {room, static_cast<uint64_t>(s.padded_columns) * parts_of(a), s.padded_columns};
}

EntropyNarrowArgs narrow_args(const EntropyArgs& a, const Saved& s) {
    EntropyNarrowArgs p{};
    p.packed = s.packed;
    p.packed_stride = s.padded_columns;
    p.table = a.table;
    p.table_stride = a.table_stride;
    p.table_rows = a.rows;
    p.columns = a.columns;
    p.padded = s.padded;
    p.count = s.count;
    p.target = s.target;
    p.lse = s.lse;
    p.to_log2 = a.scale * log2_e;
    return p;
}

// Whether a row's own target's gradient goes apart, in the table's gradient: of 16-bit types what its rounding lost, always, as the roundings of many rows of one
// target may be all alike (a table of zeros). With 64 and more rows of each target that takes 1 to 8 % of a pass, 13 where all are of one (200,000 x 300 x 200 bfloat16
// 526 -> 554 us, error of the table's gradient 0.00187 -> 0.00169, of one rounding 0.00166), a fifth against a table of one tile (100,000 x 16 x 128 142 -> 172). Of
// floats, which lose nothing, all of it, where no table row is the target of more than 64 on average (rows left out
// among them: how many count is known on the device alone): past that the rows to look up are as many as those of a product's steps.
bool targets_apart(const EntropyArgs& a) { return !in_parts(a) || a.n / 64 <= a.rows; }

// of a slab's first `rows` rows, as they lie
Gathering gathering_of(const float* slab, uint64_t slab_rows, uint32_t slab_stride, uint32_t splits, uint32_t rows, uint32_t columns, const float* factor) {
    Gathering g{};
    g.slab = slab;
    g.slab_rows = slab_rows;
    g.slab_stride = slab_stride;
    g.splits = splits;
    g.rows = rows;
    g.columns = columns;
    g.factor = factor;
    return g;
}

void launch_gathering(int type, const Gathering& g, void* out, hipStream_t stream) {
    if (g.rows == 0 || g.columns == 0) return;
    const uint64_t items = static_cast<uint64_t>(g.rows) * ((g.columns + 3) / 4);
    const uint32_t blocks = copy_grid(items);
    with_type(type, [&](auto t) {
        using T = decltype(t);
        if (g.splits >= 16 && items <= 1u << 18)
            hipLaunchKernelGGL(entropy_gather_splits_kernel<T>, dim3(div_up(items, 16)), dim3(256), 0, stream, g, static_cast<T*>(out));
        else hipLaunchKernelGGL(entropy_gather_kernel<T>, dim3(blocks), dim3(256), 0, stream, g, static_cast<T*>(out));
    });
}

bool launch_narrow_backward(const EntropyArgs& a, const float* upstream, const Saved& s, void* grad_features, void* grad_table, void* scratch,
                            hipStream_t stream) {
    const NarrowBackwardScratch w(a, s, scratch);
    const WeightArgs weights{upstream, s.count, s.row_of, s.padded, a.each, a.mean, a.scale, 1.0f, w.weight, w.factor};
    hipLaunchKernelGGL(entropy_weights_kernel, dim3(div_up(s.padded, 256)), dim3(256), 0, stream, weights);
    EntropyNarrowArgs p = narrow_args(a, s);
    p.weight = w.weight;
    p.slab = w.slab;
    p.slab_stride = w.slab_stride;
    if (grad_features) {
        p.slab_rows = s.padded;
        if (a.rows > 0) launch_entropy_narrow(entropy_features_gradient, a.type, p, w.features, stream);
        Gathering g = gathering_of(w.slab, s.padded, w.slab_stride, w.features.splits, a.n, a.columns, w.factor);
        g.packed_of = s.packed_of;
        g.weight = w.weight;
        launch_gathering(a.type, g, grad_features, stream);
    }
    if (grad_table) {
        p.slab_rows = a.rows;
        launch_entropy_narrow(entropy_table_gradient, a.type, p, w.table, stream);
        launch_gathering(a.type, gathering_of(w.slab, a.rows, w.slab_stride, w.table.splits, a.rows, a.columns, w.factor), grad_table, stream);
    }
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

}  // namespace

bool entropy_fits(const EntropyArgs& a) {
    const Saved s(a, nullptr);
    const uint64_t row_tiles = s.padded / tile, column_tiles = div_up(std::max(a.columns, 1u), tile);
    const uint64_t most_tiles = std::max<uint64_t>(row_tiles, div_up(a.rows, tile));
    return most_tiles * std::max<uint64_t>(column_tiles, row_tile / tile) <= most_blocks;
}

size_t entropy_saved_bytes(const EntropyArgs& a) { return Saved(a, nullptr).bytes; }
size_t entropy_forward_bytes(const EntropyArgs& a, bool backward) {
    if (!backward && few(a)) return entropy_few_bytes(a);
    const Saved s(a, nullptr);
    return (backward ? 0 : s.bytes) + ForwardScratch(a, s, nullptr).bytes;
}
size_t entropy_backward_bytes(const EntropyArgs& a) {
    return narrow(a) ? NarrowBackwardScratch(a, Saved(a, nullptr), nullptr).bytes : BackwardScratch(a, Saved(a, nullptr), nullptr).bytes;
}

bool launch_entropy_forward(const EntropyArgs& a, float* loss, void* saved, void* scratch, hipStream_t stream) {
    if (!saved && few(a)) {
        launch_entropy_few(a, loss, scratch, stream);
        EFGS_HIP_CHECK(hipGetLastError());
        return true;
    }
    const Saved s(a, saved ? saved : scratch);
    const ForwardScratch f(a, s, saved ? scratch : static_cast<char*>(scratch) + s.bytes);
    launch_packing(a, s, f.chunk_counts, stream);
    const Table table = table_of(a, s, f.copied ? f.copy : nullptr, stream);
    for (uint32_t first = 0; first < s.padded; first += f.rows_at_once) {
        const uint32_t rows = std::min(s.padded - first, f.rows_at_once);
        if (a.rows > 0 && narrow(a)) {
            EntropyNarrowArgs p = narrow_args(a, s);
            p.partial = f.partial;
            p.target_logit = f.target_logit;
            launch_entropy_narrow(entropy_logits, a.type, p, f.plan, stream);
        } else if (a.rows > 0) {
            EntropyProductArgs p{};
            p.a = table.rows;
            p.a_stride = table.stride;
            p.a_columns = table.columns * parts_of(a);
            p.a_plane = table.columns;
            p.b = s.packed;
            p.b_stride = static_cast<uint64_t>(s.padded_columns) * parts_of(a);
            p.b_plane = s.padded_columns;
            p.i_end = a.rows;
            p.j_end = rows;
            p.k_end = table.columns;
            p.i_tiles = f.tiles;
            p.j_first = first;
            p.splits = 1;
            p.count = s.count;
            p.to_log2 = a.scale * log2_e;
            p.partial = f.partial;
            p.slab_rows = rows;
            p.target_logit = f.target_logit;
            p.target = s.target;
            launch_entropy_wide(entropy_logits, a.type, f.side, p, rows, stream);
        }
        const JoinArgs j{f.partial, f.tiles, first, rows, a.n, s.count, s.row_of, s.packed_of, f.target_logit, s.lse, a.each ? loss : nullptr, f.sums};
        if (f.tiles <= join_alone) hipLaunchKernelGGL(entropy_join_kernel<1>, dim3(rows / 256), dim3(256), 0, stream, j);
        else hipLaunchKernelGGL(entropy_join_kernel<join_parts>, dim3(rows / join_rows), dim3(join_rows * join_parts), 0, stream, j);
    }
    if (!a.each) hipLaunchKernelGGL(entropy_total_kernel, dim3(1), dim3(total_block), 0, stream, f.sums, s.padded / join_rows, s.count, a.mean, loss);
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

bool launch_entropy_backward(const EntropyArgs& a, const float* upstream, const void* saved, void* grad_features, void* grad_table, void* scratch,
                             hipStream_t stream) {
    if (a.columns == 0) return true;
    const Saved s(a, const_cast<void*>(saved));
    if (narrow(a)) return launch_narrow_backward(a, upstream, s, grad_features, grad_table, scratch, stream);
    const BackwardScratch w(a, s, scratch);
    const Table table = table_of(a, s, w.copied ? w.copy : nullptr, stream);
    const bool half = a.type == type_half;
    const WeightArgs weights{upstream, s.count, s.row_of, s.padded, a.each, a.mean, a.scale, half ? entropy_half_range : 1.0f, w.weight, w.factor};
    if (half && a.each) hipLaunchKernelGGL(entropy_half_weights_kernel, dim3(1), dim3(1024), 0, stream, weights);
    else hipLaunchKernelGGL(entropy_weights_kernel, dim3(div_up(s.padded, 256)), dim3(256), 0, stream, weights);
    const uint32_t parts = parts_of(a);
    const bool apart = targets_apart(a);
    for (uint32_t piece = 0; piece < w.pieces && a.rows > 0; piece++) {
        const uint32_t first = piece * w.piece_rows, rows = std::min(a.rows - first, w.piece_rows);
        const void* const part = static_cast<const char*>(table.rows) + first * table.stride * (in_parts(a) ? 2 : type_bytes(a.type));
        EntropyProductArgs p{};
        p.a = part;
        p.a_stride = table.stride;
        p.a_columns = table.columns * parts;
        p.a_plane = table.columns;
        p.b = s.packed;
        p.b_stride = static_cast<uint64_t>(s.padded_columns) * parts;
        p.b_plane = s.padded_columns;
        p.i_end = rows;
        p.j_end = s.padded;
        p.k_end = table.columns;
        p.i_tiles = div_up(rows, w.upstream.side);
        p.splits = 1;
        p.count = s.count;
        p.to_log2 = a.scale * log2_e;
        p.target = s.target;
        p.lse = s.lse;
        p.weight = w.weight;
        p.first_row = first;
        p.piece = w.piece;
        p.residual = w.residual;
        p.apart = apart;
        p.piece_stride = static_cast<uint64_t>(w.piece_rows) * parts;
        p.piece_plane = w.piece_rows;
        launch_entropy_wide(entropy_upstream, a.type, w.upstream.side, p, s.padded, stream);
        EntropyProductArgs x{};
        x.count = s.count;
        x.i_end = a.columns;
        x.slab_stride = s.padded_columns;
        x.b = w.piece;
        x.b_stride = p.piece_stride;
        x.b_plane = w.piece_rows;
        x.target = s.target;
        x.first_row = first;
        x.residual = w.residual;
        x.apart = apart;
        if (grad_features) {
            x.a = part;
            x.a_stride = table.stride;
            x.a_columns = x.a_plane = table.columns;
            x.i_tiles = div_up(a.columns, w.features.side);
            x.j_end = s.padded;
            x.k_end = rows;
            x.splits = w.features.splits;
            x.slab = w.features_slab;
            x.slab_rows = s.padded;
            x.add = piece > 0;
            launch_entropy_wide(entropy_features_gradient, a.type, w.features.side, x, s.padded, stream);
        }
        if (grad_table) {
            void* const out = static_cast<char*>(grad_table) + static_cast<uint64_t>(first) * a.columns * type_bytes(a.type);
            x.a = s.packed;
            x.a_stride = p.b_stride;
            x.a_columns = x.a_plane = s.padded_columns;
            x.i_tiles = div_up(a.columns, w.table.side);
            x.j_end = rows;
            x.splits = w.table.splits;
            x.slab = w.table_slab;
            x.slab_rows = w.piece_rows;
            x.add = false;
            x.out = x.splits > 1 ? nullptr : out;
            x.out_stride = a.columns;
            x.factor = w.factor;
            launch_entropy_wide(entropy_table_gradient, a.type, w.table.side, x, rows, stream);
            if (x.splits > 1)
                launch_gathering(a.type, gathering_of(w.table_slab, w.piece_rows, s.padded_columns, x.splits, rows, a.columns, w.factor), out, stream);
        }
    }
    if (grad_features) {
        Gathering g = gathering_of(w.features_slab, s.padded, s.padded_columns, w.features.splits, a.n, a.columns, w.factor);
        g.packed_of = s.packed_of;
        g.residual = in_parts(a) && !apart ? nullptr : w.residual;
        g.target = s.target;
        g.table = in_parts(a) ? a.table : table.rows;
        g.table_stride = in_parts(a) ? a.table_stride : table.stride;
        launch_gathering(a.type, g, grad_features, stream);
    }
    EFGS_HIP_CHECK(hipGetLastError());
    return true;
}

}  // namespace efgs
